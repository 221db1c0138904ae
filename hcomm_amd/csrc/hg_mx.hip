// hg_mx.hip - messages in microscaled 4-bit floating point: quantising a matrix, folding k ranks' quantised messages.
//
// A block is 32 elements of a row under one power-of-two scale, 16 bytes of elements and one of scale.  Both kernels
// give a lane eight elements - one dword of packed elements - and a block four neighbouring lanes, which find the
// block's largest magnitude among themselves (two lane exchanges inside the quad, no LDS).  Both are bound by memory once
// there is enough of it (medians of the kernels' durations): 67.1M bf16 elements are quantised in 29.4 us (170 MB, 5.8 TB/s) and
// turned back in 25.1; the fold of seven ranks' 14.3M elements into fp32 takes 22.4 us (110 MB, 4.9 TB/s), that of 8.4M onto an
// addend, dense and quantised again, 18.0 us (69 MB, 3.8 TB/s: a conversion for every pair of elements and rank, and fp64 sums,
// show).  8 x 16,384 elements: 4.5 us, the latency of a launch, two loads and a store.
#include "hg_ops_device.hpp"

namespace {

// ---- where a lane's group lies ------------------------------------------------------------------------------
//
// ONE: every workgroup lies in one row, so that the row and where the workgroup begins in it are scalars and a lane adds
// a small distance of its own; otherwise a workgroup takes several short rows and the row is the lane's.

template <bool ONE> struct Place {
    uint64_t row;
    uint32_t tile;  // first group of the workgroup in its row (ONE) or 0
    uint32_t group; // of the row, from `tile` on
    bool there;
};

template <bool ONE, uint32_t U> __device__ __forceinline__ Place<ONE> place_of(const HgMxGrid& g, uint32_t u)
{
    const uint32_t wg = blockIdx.x, q = u * 256u + threadIdx.x;
    Place<ONE> p;
    if (ONE) {
        const uint32_t row = g.rows == 1u ? 0u : wg / g.tiles;
        p.row = row;
        p.tile = (wg - row * g.tiles) * (256u * U);
        p.group = q;
        p.there = q < g.groups - p.tile;
    } else {
        // q / groups by a multiplication: with q < 2^10 and 4 <= groups < 2^10 the factor rounded up to 2^-20 is exact
        const uint32_t r = (q * (((1u << 20) + g.groups - 1u) / g.groups)) >> 20;
        p.row = (uint64_t)wg * g.rows_per_wg + r;
        p.tile = 0u;
        p.group = q - r * g.groups;
        p.there = r < g.rows_per_wg && p.row < g.rows;
    }
    return p;
}

// Eight elements of a dense matrix at a place, and where they go back.  What is quantised and the dense results pass by
// the caches: 67.1M bf16 elements quantised 39 -> 28 us, 14.3M fp32 results of seven ranks 29 -> 23.
template <int DT, bool NT, bool ONE> __device__ __forceinline__ Raw8<DT> ask_at(const void* m, uint64_t stride, const Place<ONE>& p, uint64_t cols)
{
    const uint64_t at = (uint64_t)p.tile * 8u;
    return ask8<DT, true, NT>((const uint8_t*)m + (p.row * stride + at) * ElemSize<DT>::v, p.group * 8u, p.there ? cols - at : 0u, cols < 8u);
}
template <int DT, bool ONE> __device__ __forceinline__ void settle_at(Raw8<DT>& v, const Place<ONE>& p, uint64_t cols)
{
    settle8<DT, true>(v, p.group * 8u, p.there ? cols - (uint64_t)p.tile * 8u : 0u, cols < 8u);
}
template <int DT, bool ONE> __device__ __forceinline__ void store_at(void* m, uint64_t stride, const Place<ONE>& p, uint64_t cols, const Raw8<DT>& v)
{
    const uint64_t at = (uint64_t)p.tile * 8u;
    store8<DT, true, true>((uint8_t*)m + (p.row * stride + at) * ElemSize<DT>::v, p.group * 8u, p.there ? cols - at : 0u, v);
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

template <bool ONE> __device__ __forceinline__ void put_group(const HgMxView& out, const Place<ONE>& p, uint32_t w, uint32_t s)
{
    uint8_t* packed = out.packed + (p.row * out.packed_stride + (uint64_t)p.tile * 4u);
    uint8_t* scales = out.scales + (p.row * out.scale_stride + (p.tile >> 2));
    *(__attribute__((address_space(1))) uint32_t*)(packed + p.group * 4u) = w;
    if ((p.group & 3u) == 0u) ((__attribute__((address_space(1))) uint8_t*)scales)[p.group >> 2] = (uint8_t)s;
}

// ---- quantise ---------------------------------------------------------------------------------------------------

template <int DT, bool ONE, uint32_t U> __global__ __launch_bounds__(256) void k_mx_quantize(const HgMxQuantize a)
{
    Raw8<DT> x[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) x[u] = ask_at<DT, true>(a.src, a.src_stride, place_of<ONE, U>(a.grid, u), a.grid.cols);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const Place<ONE> p = place_of<ONE, U>(a.grid, u);
        float f[8];
        settle_at(x[u], p, a.grid.cols);
        widen8<DT>(x[u], f);
        uint32_t m = 0;
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) {
            const uint32_t b = f32_bits(f[e]) & 0x7fffffffu;
            m = b > m ? b : m;
        }
        const uint32_t s = scale_of(quad_max(m));
        if (p.there) put_group(a.out, p, encode8(f, s), s);
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

// fp64 to fp32, rounded to odd: what a further rounding to fewer bits makes of it is what it would make of the fp64 value.
// A finite value past fp32's range becomes fp32's largest number, whose last bit is odd: infinite in a narrower dense type, and
// in a block elements under the largest scale that fp32 numbers have.
__device__ __forceinline__ float to_odd(double v)
{
    float f = (float)v;
    const double back = (double)f;
    uint32_t u = f32_bits(f);
    if (back != v && (u & 0x7fffffffu) <= 0x7f800000u && !(u & 1u)) u += (__builtin_fabs(v) > __builtin_fabs(back)) ? 1u : 0xffffffffu;
    return bits_f32(u);
}

__device__ __forceinline__ void decode8(uint32_t w, float sc, float (&f)[8])
{
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 3);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = c.x, f[5] = c.y, f[6] = d.x, f[7] = d.y;
}

// The arguments as the kernel takes them: the runtime copies them at every launch, so a fold of few ranks carries few views.
template <uint32_t N> struct FoldArgs {
    HgMxGrid grid;
    HgMxView src[N];
    HgMxView again;
    void* dst;
    const void* addend;
    uint64_t dst_stride, addend_stride;
    uint32_t k;
};

// the fp64 sum of the ranks' values from `to` on, or of the ranks' values alone where nothing is there yet
template <uint32_t B> __device__ __forceinline__ void fold_wide(double (&to)[8], bool empty, const uint32_t (&w)[B], const uint32_t (&s)[B], uint32_t n)
{
    for (uint32_t j = 0; j < n; ++j) {
        uint32_t wj = w[0], sj = s[0];
#pragma unroll
        for (uint32_t i = 1; i < B; ++i) wj = i == j ? w[i] : wj, sj = i == j ? s[i] : sj;
        float x[8];
        decode8(wj, scale_f32(sj), x);
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) to[e] = empty && j == 0u ? (double)x[e] : to[e] + (double)x[e];
    }
}

// JOIN: there is an addend or there are more than eight ranks, so that fp64 has to join exact sums
template <int DT, bool ONE, uint32_t N, bool JOIN> __global__ __launch_bounds__(256) void k_mx_reduce(const FoldArgs<N> a)
{
    constexpr uint32_t B = N < FOLD_BATCH ? N : FOLD_BATCH;
    const Place<ONE> p = place_of<ONE, 1>(a.grid, 0u);
    double v[8];             // JOIN: the sum
    float odd[8], near[8];   // the sum as what narrower types round it from, and rounded to fp32
    Raw8<DT> own;
    if (JOIN && a.addend) own = ask_at<DT, false>(a.addend, a.addend_stride, p, a.grid.cols);
    for (uint32_t j0 = 0; j0 < (JOIN ? a.k : 1u); j0 += B) {
        uint32_t w[B], s[B];
        const uint32_t n = N == 1u ? 1u : min(a.k - j0, B);
#pragma unroll
        for (uint32_t j = 0; j < B; ++j) {
            w[j] = 0u, s[j] = 127u;
            if (j < n && p.there) {
                const HgMxView& r = a.src[j0 + j];
                const uint8_t* packed = r.packed + (p.row * r.packed_stride + (uint64_t)p.tile * 4u);
                const uint8_t* scales = r.scales + (p.row * r.scale_stride + (p.tile >> 2));
                w[j] = *(const __attribute__((address_space(1))) uint32_t*)(packed + p.group * 4u);
                s[j] = ((const __attribute__((address_space(1))) uint8_t*)scales)[p.group >> 2];
            }
        }
        const bool empty = !JOIN || (j0 == 0u && !a.addend);
        if (JOIN && j0 == 0u && a.addend) {
            float x[8];
            settle_at(own, p, a.grid.cols);
            widen8<DT>(own, x);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) v[e] = (double)x[e];
        }
        uint32_t lo = 255u, hi = 0u; // scales that have a nonzero element under them
#pragma unroll
        for (uint32_t j = 0; j < B; ++j) {
            const bool any = (w[j] & 0x77777777u) != 0u || s[j] == 255u;
            lo = any && s[j] < lo ? s[j] : lo;
            hi = any && s[j] > hi ? s[j] : hi;
        }
        if (N == 1u || !(hi > lo + 17u || hi > 240u)) {
            float f[8];
            decode8(w[0], scale_f32(s[0]), f);
#pragma unroll
            for (uint32_t j = 1; j < B; ++j)
                if (j < n) {
                    float x[8];
                    decode8(w[j], scale_f32(s[j]), x);
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e) f[e] += x[e];
                }
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) {
                if (JOIN) v[e] = empty ? (double)f[e] : v[e] + (double)f[e];
                else odd[e] = near[e] = f[e];
            }
        } else if (JOIN) {
            fold_wide(v, empty, w, s, n);
        } else {
            double x[8];
            fold_wide(x, true, w, s, n);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) odd[e] = to_odd(x[e]), near[e] = (float)x[e];
        }
    }
    if (JOIN) {
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) odd[e] = to_odd(v[e]), near[e] = (float)v[e];
    }
    if (a.dst) store_at<DT>(a.dst, a.dst_stride, p, a.grid.cols, DT == DT_F32 ? narrow8<DT>(near) : narrow8<DT>(odd));
    if (a.again.packed) {
        const int64_t left = (int64_t)(a.grid.cols - ((uint64_t)p.tile + p.group) * 8u); // elements to the row's end
        uint32_t m = 0;
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) {
            if (left <= (int64_t)e) odd[e] = 0.0f; // elements past it do not count, whatever the inputs hold there
            const uint32_t b = f32_bits(odd[e]) & 0x7fffffffu;
            m = b > m ? b : m;
        }
        const uint32_t s = scale_of(quad_max(m));
        if (p.there) put_group(a.again, p, encode8(odd, s), s);
    }
}

template <class K, class A> int launch(hipStream_t st, uint32_t wgs, K kernel, const A& a)
{
    hipLaunchKernelGGL(kernel, dim3(wgs), dim3(256), 0, st, a);
    return rc(hipGetLastError());
}

template <int DT> int quantize(hipStream_t st, const HgMxQuantize& a)
{
    const bool one = a.grid.rows_per_wg == 1u;
    if (a.grid.tile == 256u) return one ? launch(st, a.grid.wgs, k_mx_quantize<DT, true, 1>, a) : launch(st, a.grid.wgs, k_mx_quantize<DT, false, 1>, a);
    return one ? launch(st, a.grid.wgs, k_mx_quantize<DT, true, HG_MX_UNROLL>, a) : launch(st, a.grid.wgs, k_mx_quantize<DT, false, HG_MX_UNROLL>, a);
}

template <int DT, uint32_t N, bool JOIN> int reduce_n(hipStream_t st, const HgMxReduce& a)
{
    FoldArgs<N> f;
    f.grid = a.grid;
    for (uint32_t j = 0; j < N; ++j) f.src[j] = a.src[j];
    f.again = a.again;
    f.dst = a.dst, f.addend = a.addend, f.dst_stride = a.dst_stride, f.addend_stride = a.addend_stride, f.k = a.k;
    return a.grid.rows_per_wg > 1u ? launch(st, a.grid.wgs, k_mx_reduce<DT, false, N, JOIN>, f) : launch(st, a.grid.wgs, k_mx_reduce<DT, true, N, JOIN>, f);
}

template <int DT> int reduce(hipStream_t st, const HgMxReduce& a)
{
    if (a.k > FOLD_BATCH) return reduce_n<DT, HCOMM_GFX_MAX_RANKS, true>(st, a);
    if (a.addend) return reduce_n<DT, FOLD_BATCH, true>(st, a);
    return a.k == 1u ? reduce_n<DT, 1, false>(st, a) : reduce_n<DT, FOLD_BATCH, false>(st, a);
}

} // namespace

extern "C" {

int hg_launch_mx_quantize(void* stream, const void* args)
{
    const HgMxQuantize* a = (const HgMxQuantize*)args;
    OnDeviceOf device((hipStream_t)stream);
    if (device.err != hipSuccess) return HCCL_E_RUNTIME;
    switch (a->dtype) {
        case DT_F16: return quantize<DT_F16>((hipStream_t)stream, *a);
        case DT_BF16: return quantize<DT_BF16>((hipStream_t)stream, *a);
        case DT_F32: return quantize<DT_F32>((hipStream_t)stream, *a);
        default: return HCCL_E_PARA;
    }
}

int hg_launch_mx_reduce(void* stream, const void* args)
{
    const HgMxReduce* a = (const HgMxReduce*)args;
    OnDeviceOf device((hipStream_t)stream);
    if (device.err != hipSuccess) return HCCL_E_RUNTIME;
    switch (a->dtype) {
        case DT_F16: return reduce<DT_F16>((hipStream_t)stream, *a);
        case DT_BF16: return reduce<DT_BF16>((hipStream_t)stream, *a);
        case DT_F32: return reduce<DT_F32>((hipStream_t)stream, *a);
        default: return HCCL_E_PARA;
    }
}

} // extern "C"
