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
typedef uint32_t u32x2_raw __attribute__((ext_vector_type(2)));
typedef u32x2_raw __attribute__((aligned(2))) u32x2_at2;
typedef u32x2_raw __attribute__((aligned(4))) u32x2_at4;
typedef uint32_t __attribute__((aligned(2))) u32_at2;
// eight elements in one or two accesses; four, two and one of them
template <int DT> struct GroupVec {
    typedef u32x4_at2 type;
    typedef u32x2_at2 half;
    typedef u32_at2 quarter;
    typedef uint16_t eighth;
    static __device__ __forceinline__ uint32_t pair(const uint32_t* w) { return w[0]; }
};
template <> struct GroupVec<DT_F32> {
    typedef u32x4_at4 type;
    typedef u32x4_at4 half;
    typedef u32x2_at4 quarter;
    typedef uint32_t eighth;
    static __device__ __forceinline__ u32x2_raw pair(const uint32_t* w) { return u32x2_raw{w[0], w[1]}; }
};

// Elements [at, at + 8) of a row of which `cols` are left; those past its end are 0.  TAIL: a row may end inside a group of
// eight; without it a group is there or not.  NT: a cache hint for what is read (written) once and by no launch that follows
// soon.  A group that the row's end cuts is read as the row's last eight elements, which settle8, called where the group is
// used, moves to where they belong: no load waits for another.  `short_row`: the whole row has fewer than eight (uniform).
// ask8_into: where a row ends before the group, what was there stays (a buffer that is used again needs its zeros once).
// Here and in store8 `at` counts from `row` in 32 bits of bytes: in a row that may be longer, `row` is a place near the group.
template <int DT, bool TAIL, bool NT> __device__ __forceinline__ void ask8_into(Raw8<DT>& r, const void* row, uint32_t at, uint64_t cols, bool short_row)
{
    constexpr uint32_t ES = ElemSize<DT>::v, W = Raw8<DT>::words;
    typedef const __attribute__((address_space(1))) typename GroupVec<DT>::type cv;
    if (TAIL && short_row) {
#pragma unroll
        for (uint32_t i = 0; i < W; ++i) r.w[i] = 0u;
        // from the last element on, each moves those behind it up by one place
#pragma unroll 1
        for (uint32_t e = at == 0u ? (uint32_t)cols : 0u; e-- != 0u;) {
            const uint32_t x = ld_elem<ES>((const uint8_t*)row + e * ES);
#pragma unroll
            for (uint32_t i = W; i-- != 0u;) {
                const uint32_t below = i ? r.w[i ? i - 1u : 0u] : 0u;
                r.w[i] = ES == 4u ? (i ? below : x) : (r.w[i] << 16) | (i ? below >> 16 : x);
            }
        }
        return;
    }
    if (at < cols) {
        const int32_t back = TAIL && at + 8u > cols ? (int32_t)(at + 8u - (uint32_t)cols) : 0; // may reach in front of `row`, not of the whole row
        const uint8_t* p = (const uint8_t*)row + (int64_t)((int32_t)at - back) * (int32_t)ES;
#pragma unroll
        for (uint32_t i = 0; i < W / 4u; ++i) {
            const u32x4 v = NT ? __builtin_nontemporal_load((cv*)p + i) : ((cv*)p)[i];
            r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
        }
    }
}
template <int DT> __device__ __forceinline__ Raw8<DT> zeros8()
{
    Raw8<DT> r;
#pragma unroll
    for (uint32_t i = 0; i < Raw8<DT>::words; ++i) r.w[i] = 0u;
    return r;
}
template <int DT, bool TAIL, bool NT> __device__ __forceinline__ Raw8<DT> ask8(const void* row, uint32_t at, uint64_t cols, bool short_row)
{
    Raw8<DT> r = zeros8<DT>();
    ask8_into<DT, TAIL, NT>(r, row, at, cols, short_row);
    return r;
}

template <int DT, bool TAIL> __device__ __forceinline__ void settle8(Raw8<DT>& r, uint32_t at, uint64_t cols, bool short_row)
{
    if (!TAIL || short_row || at >= cols || at + 8u <= cols) return;
    const uint32_t by = (at + 8u - (uint32_t)cols) * ElemSize<DT>::v; // bytes that lie in front
    constexpr uint32_t W = Raw8<DT>::words;
#pragma unroll
    for (uint32_t step = 1; step < W; step *= 2u)
#pragma unroll
        for (uint32_t i = 0; i < W; ++i) {
            const uint32_t from = i + step < W ? r.w[i + step < W ? i + step : i] : 0u;
            r.w[i] = (by & (4u * step)) ? from : r.w[i];
        }
    if (ElemSize<DT>::v == 2u && (by & 2u)) {
#pragma unroll
        for (uint32_t i = 0; i < W; ++i) r.w[i] = (r.w[i] >> 16) | (i + 1u < W ? r.w[i + 1u < W ? i + 1u : i] << 16 : 0u);
    }
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
        // four, two and one elements as the count asks for them, the rest moved up behind each
        typedef __attribute__((address_space(1))) typename GroupVec<DT>::half wh;
        typedef __attribute__((address_space(1))) typename GroupVec<DT>::quarter wq;
        typedef __attribute__((address_space(1))) typename GroupVec<DT>::eighth we;
        const uint32_t n = (uint32_t)(cols - at);
        constexpr uint32_t H = Raw8<DT>::words / 2u, Q = H / 2u;
        uint32_t w[H];
#pragma unroll
        for (uint32_t i = 0; i < H; ++i) w[i] = r.w[i];
        if (n & 4u) {
            typename GroupVec<DT>::half v;
#pragma unroll
            for (uint32_t i = 0; i < H; ++i) v[i] = w[i], w[i] = r.w[H + i];
            *(wh*)p = v;
            p += 4u * ES;
        }
        if (n & 2u) {
            *(wq*)p = GroupVec<DT>::pair(w);
            p += 2u * ES;
#pragma unroll
            for (uint32_t i = 0; i < Q; ++i) w[i] = w[Q + i];
        }
        if (n & 1u) *(we*)p = (typename GroupVec<DT>::eighth)w[0];
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
