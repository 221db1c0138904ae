// hg_ops_device.hpp - what the operators around a fold share on the device: eight elements of a row at a time, widened
// to fp32 and rounded back once.
#pragma once
#include "hg_device.hpp"
#include "hg_ops.h"

namespace {

// Eight elements as they lie in memory.  Rows start at any element, so a full group is one or two 128-bit accesses
// that need not be aligned to more than the element (the target takes those; on aligned rows they cost nothing).
template <int DT> struct Raw8 {
    static constexpr uint32_t words = (DT == DT_F32) ? 8u : 4u;
    uint32_t w[words];
};

typedef u32x4 __attribute__((aligned(2))) u32x4_at2;
typedef u32x4 __attribute__((aligned(4))) u32x4_at4;
template <int DT> struct GroupVec { typedef u32x4_at2 type; };
template <> struct GroupVec<DT_F32> { typedef u32x4_at4 type; };

// Elements [at, at + 8) of a row that holds `cols`; those past its end are 0.  TAIL: a row may end inside a group of eight;
// without it a group is there or not, and a load is one predicate and no branch of its own.  NT: a cache hint for what
// is read (written) once and by no launch that follows soon.
template <int DT, bool TAIL = true, bool NT = false> __device__ __forceinline__ Raw8<DT> load8(const void* row, uint32_t at, uint64_t cols)
{
    constexpr uint32_t ES = ElemSize<DT>::v;
    typedef const __attribute__((address_space(1))) typename GroupVec<DT>::type cv;
    Raw8<DT> r;
    const uint8_t* p = (const uint8_t*)row + at * ES;
    if (TAIL ? at + 8u <= cols : at < cols) {
#pragma unroll
        for (uint32_t i = 0; i < Raw8<DT>::words / 4u; ++i) {
            const u32x4 v = NT ? __builtin_nontemporal_load((cv*)p + i) : ((cv*)p)[i];
            r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < Raw8<DT>::words; ++i) r.w[i] = 0u;
        if (TAIL && at < cols) {
            const uint32_t n = (uint32_t)(cols - at);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e)
                if (e < n) {
                    const uint32_t x = ld_elem<ES>(p + e * ES);
                    if (ES == 4) r.w[e] = x;
                    else r.w[e / 2u] |= x << (16u * (e % 2u));
                }
        }
    }
    return r;
}

template <int DT> __device__ __forceinline__ void widen8(const Raw8<DT>& r, float (&f)[8])
{
#pragma unroll
    for (uint32_t e = 0; e < 8u; ++e) {
        if (DT == DT_F32) f[e] = bits_f32(r.w[e]);
        else if (DT == DT_BF16) f[e] = bits_f32((e % 2u) ? (r.w[e / 2u] & 0xffff0000u) : (r.w[e / 2u] << 16));
        else {
            const f16x2 h = __builtin_bit_cast(f16x2, r.w[e / 2u]);
            f[e] = (float)((e % 2u) ? h.y : h.x);
        }
    }
}

// round to nearest, ties to even: the one rounding of an output
template <int DT> __device__ __forceinline__ Raw8<DT> narrow8(const float (&f)[8])
{
    Raw8<DT> r;
#pragma unroll
    for (uint32_t i = 0; i < Raw8<DT>::words; ++i) {
        if (DT == DT_F32) r.w[i] = f32_bits(f[i]);
        else {
            const f32x2 v = {f[(2u * i) % 8u], f[(2u * i + 1u) % 8u]};
            if (DT == DT_BF16) r.w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
            else r.w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
        }
    }
    return r;
}

template <int DT, bool TAIL = true, bool NT = false> __device__ __forceinline__ void store8(void* row, uint32_t at, uint64_t cols, const Raw8<DT>& r)
{
    constexpr uint32_t ES = ElemSize<DT>::v;
    typedef __attribute__((address_space(1))) typename GroupVec<DT>::type wv;
    uint8_t* p = (uint8_t*)row + at * ES;
    if (TAIL ? at + 8u <= cols : at < cols) {
#pragma unroll
        for (uint32_t i = 0; i < Raw8<DT>::words / 4u; ++i) {
            const typename GroupVec<DT>::type v = u32x4{r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]};
            if (NT) __builtin_nontemporal_store(v, (wv*)p + i);
            else ((wv*)p)[i] = v;
        }
    } else if (TAIL && at < cols) {
        const uint32_t n = (uint32_t)(cols - at);
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e)
            if (e < n) st_elem<ES>(p + e * ES, ES == 4 ? r.w[e % Raw8<DT>::words] : (r.w[e / 2u] >> (16u * (e % 2u))) & 0xffffu);
    }
}

// The launch goes to the stream's own device (the default stream: the current one), which need not be current.
struct OnDeviceOf {
    int before = -1;
    hipError_t err = hipSuccess;
    explicit OnDeviceOf(hipStream_t stream)
    {
        hipDevice_t d = 0;
        int cur = -1;
        if (!stream) return;
        err = hipStreamGetDevice(stream, &d);
        if (err == hipSuccess) err = hipGetDevice(&cur);
        if (err == hipSuccess && (int)d != cur) {
            err = hipSetDevice((int)d);
            if (err == hipSuccess) before = cur;
        }
    }
    ~OnDeviceOf()
    {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

} // namespace
