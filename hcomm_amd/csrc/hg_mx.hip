// hg_mx.hip - messages in microscaled 4-bit floating point: quantising a matrix, folding k ranks' quantised messages.
//
// A block is 32 elements of a row under one power-of-two scale, 16 bytes of elements and one of scale.  Both kernels
// give a lane eight elements - one dword of packed elements - and a block four neighbouring lanes, which find the
// block's largest magnitude among themselves (two lane exchanges inside the quad, no LDS).  Both are bound by memory.
#include "hg_ops_device.hpp"

namespace {

// ---- where a lane's group lies ------------------------------------------------------------------------------

struct Place {
    uint64_t row;
    uint32_t group; // of the row
    bool there;
};

__device__ __forceinline__ Place place_of(const HgMxGrid& g, uint32_t q)
{
    const uint32_t wg = blockIdx.x;
    Place p;
    if (g.rows_per_wg <= 1u) {
        const uint32_t row = wg / g.tiles, tile = wg - row * g.tiles;
        p.row = row;
        p.group = tile * HG_MX_TILE + q;
        p.there = p.group < g.groups;
    } else {
        // q / groups by a multiplication: with q < 2^10 and 2 <= groups < 2^10 the factor rounded up to 2^-20 is exact
        const uint32_t r = (q * (((1u << 20) + g.groups - 1u) / g.groups)) >> 20;
        p.row = (uint64_t)wg * g.rows_per_wg + r;
        p.group = q - r * g.groups;
        p.there = r < g.rows_per_wg && p.row < g.rows;
    }
    return p;
}

// the largest of a value over the four lanes of a block
__device__ __forceinline__ uint32_t quad_max(uint32_t v)
{
    const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true); // lanes 1 0 3 2
    v = v > a ? v : a;
    const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true); // lanes 2 3 0 1
    return v > b ? v : b;
}

// the scale byte of a block whose largest magnitude has these fp32 bits: two below its exponent, 255 for infinities and NaN
__device__ __forceinline__ uint32_t scale_of(uint32_t amax)
{
    const uint32_t e = amax >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}

// 2^(s - 127) as the conversions take it (2^-127 is subnormal); only the exponent counts there
__device__ __forceinline__ float scale_f32(uint32_t s) { return bits_f32(s ? s << 23 : 0x00400000u); }

// eight fp32 values to eight elements under scale s, nearest even, saturating (one instruction a pair)
__device__ __forceinline__ uint32_t encode8(const float (&f)[8], uint32_t s)
{
    const float sc = scale_f32(s);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0], f[1], sc, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2], f[3], sc, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4], f[5], sc, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6], f[7], sc, 3);
    return s == 255u ? 0u : w;
}

__device__ __forceinline__ void put_group(const HgMxView& out, const Place& p, uint32_t w, uint32_t s)
{
    *(__attribute__((address_space(1))) uint32_t*)(out.packed + p.row * out.packed_stride + (uint64_t)p.group * 4u) = w;
    if ((p.group & 3u) == 0u) out.scales[p.row * out.scale_stride + (p.group >> 2)] = (uint8_t)s;
}

// ---- quantise ---------------------------------------------------------------------------------------------------

template <int DT> __global__ __launch_bounds__(256) void k_mx_quantize(const HgMxQuantize a)
{
    constexpr uint32_t U = HG_MX_TILE / 256u;
    Place p[U];
    Raw8<DT> x[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        p[u] = place_of(a.grid, u * 256u + threadIdx.x);
        const uint8_t* row = (const uint8_t*)a.src + p[u].row * a.src_stride * ElemSize<DT>::v;
        x[u] = load8<DT>(row, (uint64_t)p[u].group * 8u, p[u].there ? a.grid.cols : 0u);
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        float f[8];
        widen8<DT>(x[u], f);
        uint32_t m = 0;
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) {
            const uint32_t b = f32_bits(f[e]) & 0x7fffffffu;
            m = b > m ? b : m;
        }
        const uint32_t s = scale_of(quad_max(m));
        if (p[u].there) put_group(a.out, p[u], encode8(f, s), s);
    }
}

// ---- fold ---------------------------------------------------------------------------------------------------------
//
// The sum has to be better than fp32: E2M1 values under powers of two fall on the middle between two elements all the
// time, and there the last bit of an fp32 sum would decide what the sum is quantised to.  But eight such values are
// multiples of their smallest unit 2^(smin - 128) and below 96 * 2^(smax - 128), so while smax - smin <= 17 an fp32
// sum of eight is exact (7 + 17 bits); only blocks whose ranks lie further apart are summed in fp64, and fp64 joins
// the sums of eight ranks and the addend.

constexpr uint32_t FOLD_BATCH = 8;

// fp64 to fp32, rounded to odd: what a further rounding to fewer bits makes of it is what it would make of the fp64 value
__device__ __forceinline__ float to_odd(double v)
{
    float f = (float)v;
    const double back = (double)f;
    uint32_t u = f32_bits(f);
    if (back != v && (u & 0x7f800000u) != 0x7f800000u && !(u & 1u)) u += (__builtin_fabs(v) > __builtin_fabs(back)) ? 1u : 0xffffffffu;
    return bits_f32(u);
}

__device__ __forceinline__ void decode8(uint32_t w, float sc, float (&f)[8])
{
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 3);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = c.x, f[5] = c.y, f[6] = d.x, f[7] = d.y;
}

template <int DT> __global__ __launch_bounds__(256) void k_mx_reduce(const HgMxReduce a)
{
    constexpr uint32_t U = HG_MX_TILE / 256u;
    const bool join = a.k > FOLD_BATCH || a.addend != nullptr; // more than one exact sum to add up
    for (uint32_t u = 0; u < U; ++u) {
        const Place p = place_of(a.grid, u * 256u + threadIdx.x);
        const uint64_t at = (uint64_t)p.group * 8u;
        double v[8];
        float f[8];
        bool wide = join;
        if (a.addend) {
            float x[8];
            const uint8_t* row = (const uint8_t*)a.addend + p.row * a.addend_stride * ElemSize<DT>::v;
            widen8<DT>(load8<DT>(row, at, p.there ? a.grid.cols : 0u), x);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) v[e] = (double)x[e];
        }
        for (uint32_t j0 = 0; j0 < a.k; j0 += FOLD_BATCH) {
            uint32_t w[FOLD_BATCH], s[FOLD_BATCH];
#pragma unroll
            for (uint32_t j = 0; j < FOLD_BATCH; ++j) {
                w[j] = 0u, s[j] = 127u;
                if (j0 + j < a.k && p.there) {
                    const HgMxView& r = a.src[j0 + j];
                    w[j] = *(const __attribute__((address_space(1))) uint32_t*)(r.packed + p.row * r.packed_stride + (uint64_t)p.group * 4u);
                    s[j] = ((const __attribute__((address_space(1))) uint8_t*)r.scales)[p.row * r.scale_stride + (p.group >> 2)];
                }
            }
            uint32_t lo = 255u, hi = 0u; // scales that have a nonzero element under them
#pragma unroll
            for (uint32_t j = 0; j < FOLD_BATCH; ++j) {
                const bool any = (w[j] & 0x77777777u) != 0u || s[j] == 255u;
                lo = any && s[j] < lo ? s[j] : lo;
                hi = any && s[j] > hi ? s[j] : hi;
            }
            const bool apart = hi > lo + 17u || hi > 240u;
            const bool first = j0 == 0u && !a.addend;
            if (!apart) {
                decode8(w[0], scale_f32(s[0]), f);
#pragma unroll
                for (uint32_t j = 1; j < FOLD_BATCH; ++j)
                    if (j0 + j < a.k) {
                        float x[8];
                        decode8(w[j], scale_f32(s[j]), x);
#pragma unroll
                        for (uint32_t e = 0; e < 8u; ++e) f[e] += x[e];
                    }
                if (wide) {
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e) v[e] = first ? (double)f[e] : v[e] + (double)f[e];
                }
            } else {
                wide = true;
                for (uint32_t j = 0; j < FOLD_BATCH && j0 + j < a.k; ++j) {
                    uint32_t wj = w[0], sj = s[0];
#pragma unroll
                    for (uint32_t i = 1; i < FOLD_BATCH; ++i) wj = i == j ? w[i] : wj, sj = i == j ? s[i] : sj;
                    float x[8];
                    decode8(wj, scale_f32(sj), x);
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e) v[e] = first && j == 0u ? (double)x[e] : v[e] + (double)x[e];
                }
            }
        }
        if (wide) {
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) f[e] = to_odd(v[e]);
        }
        if (a.again.packed) {
            uint32_t m = 0;
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) {
                if (at + e >= a.grid.cols) f[e] = 0.0f; // elements past the row's end do not count, whatever the inputs hold there
                const uint32_t b = f32_bits(f[e]) & 0x7fffffffu;
                m = b > m ? b : m;
            }
            const uint32_t s = scale_of(quad_max(m));
            if (p.there) put_group(a.again, p, encode8(f, s), s);
        }
        if (a.dst && p.there) {
            if (DT == DT_F32 && wide) {
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) f[e] = (float)v[e];
            }
            store8<DT>((uint8_t*)a.dst + p.row * a.dst_stride * ElemSize<DT>::v, at, a.grid.cols, narrow8<DT>(f));
        }
    }
}

template <class A, class F> int launch(void* stream, const A* a, F kernel)
{
    OnDeviceOf device((hipStream_t)stream);
    if (device.err != hipSuccess) return HCCL_E_RUNTIME;
    hipLaunchKernelGGL(kernel, dim3(a->grid.wgs), dim3(256), 0, (hipStream_t)stream, *a);
    return rc(hipGetLastError());
}

} // namespace

extern "C" {

int hg_launch_mx_quantize(void* stream, const void* args)
{
    const HgMxQuantize* a = (const HgMxQuantize*)args;
    switch (a->dtype) {
        case DT_F16: return launch(stream, a, k_mx_quantize<DT_F16>);
        case DT_BF16: return launch(stream, a, k_mx_quantize<DT_BF16>);
        case DT_F32: return launch(stream, a, k_mx_quantize<DT_F32>);
        default: return HCCL_E_PARA;
    }
}

int hg_launch_mx_reduce(void* stream, const void* args)
{
    const HgMxReduce* a = (const HgMxReduce*)args;
    switch (a->dtype) {
        case DT_F16: return launch(stream, a, k_mx_reduce<DT_F16>);
        case DT_BF16: return launch(stream, a, k_mx_reduce<DT_BF16>);
        case DT_F32: return launch(stream, a, k_mx_reduce<DT_F32>);
        default: return HCCL_E_PARA;
    }
}

} // extern "C"
