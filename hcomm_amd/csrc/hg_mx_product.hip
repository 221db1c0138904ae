// hg_mx_product.hip - the product of two matrices in microscaled 4-bit floating point, summed over the ranks that share
// its inner length: dst = sum over r of a[r] * transpose(b[r]).
//
// The matrix instruction of 16 x 16 x 128 takes the format as it is stored: lane l gives row l % 16 of an operand, 32
// consecutive elements (one block, 16 bytes) and that block's scale byte, and the four lanes of a row cover 128
// elements.  Which blocks those are is free, as long as both operands agree.  A chunk of 16 blocks of a row is given to
// its four lanes in runs of four, so that a lane's scales for four instructions are one dword of the scale row, of
// which every instruction selects its byte.
#include "hg_ops_device.hpp"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32_at1 __attribute__((aligned(1)));

#define MX_FP4 4 /* element format operand of the matrix instruction */
#define CHUNK_BLOCKS 16u

// acc += a * b for byte T of each lane's scales
template <int T> __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 acc, uint32_t sa, uint32_t sb)
{
    const i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, MX_FP4, MX_FP4, T, (int)sa, T, (int)sb);
}

// what a lane holds of one row for one chunk: four blocks and their scales
struct Run {
    u32x4 block[4];
    uint32_t scales;
};

// blocks [first, first + 4) of a row of `blocks`; those past its end are 0 under scale 1
__device__ __forceinline__ Run load_run(const HgMxView& v, uint64_t row, uint32_t first, uint32_t blocks)
{
    Run r;
    cgvec* p = (cgvec*)(v.packed + row * v.packed_stride) + first;
    const __attribute__((address_space(1))) uint8_t* s = (const __attribute__((address_space(1))) uint8_t*)(v.scales + row * v.scale_stride) + first;
    if (first + 4u <= blocks) {
#pragma unroll
        for (uint32_t t = 0; t < 4u; ++t) r.block[t] = p[t];
        r.scales = *(const __attribute__((address_space(1))) u32_at1*)s;
    } else {
        r.scales = 0x7f7f7f7fu;
#pragma unroll
        for (uint32_t t = 0; t < 4u; ++t) {
            r.block[t] = u32x4{0u, 0u, 0u, 0u};
            if (first + t < blocks) {
                r.block[t] = p[t];
                r.scales = (r.scales & ~(0xffu << (8u * t))) | ((uint32_t)s[t] << (8u * t));
            }
        }
    }
    return r;
}

// elements past `cols` do not count, whatever the last block holds there (one operand's being 0 is enough)
__device__ __forceinline__ void cut_run(Run& r, uint32_t first, uint32_t cols)
{
    const uint32_t last = (cols - 1u) / HCOMM_GFX_MX_BLOCK, n = cols - last * HCOMM_GFX_MX_BLOCK; // n elements of block `last` count
#pragma unroll
    for (uint32_t t = 0; t < 4u; ++t)
        if (first + t == last) {
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                const uint32_t keep = n > 8u * i ? n - 8u * i : 0u;
                r.block[t][i] &= keep >= 8u ? 0xffffffffu : (1u << (4u * keep)) - 1u;
            }
        }
}

__device__ __forceinline__ void put(void* dst, int dtype, uint64_t i, float v)
{
    if (dtype == DT_F32) ((__attribute__((address_space(1))) float*)dst)[i] = v;
    else if (dtype == DT_BF16) ((__attribute__((address_space(1))) __bf16*)dst)[i] = (__bf16)v;
    else ((__attribute__((address_space(1))) _Float16*)dst)[i] = (_Float16)v;
}

// ---- few rows: the operands go from memory straight into the matrix instructions --------------------------------------
//
// A workgroup owns 16 FA x 16 FB results; its four wavefronts share the inner length (chunk u of all ranks' chunks goes to
// wavefront u % 4) and add their sums up through LDS in a fixed order.
template <int FA, int FB> __global__ __launch_bounds__(256) void k_mx_product_direct(const HgMxProduct a)
{
    __shared__ f32x4 part[3][FA * FB][64];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tiles_n = (a.n + 16u * FB - 1u) / (16u * FB);
    const uint32_t tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
    const uint32_t m0 = tm * 16u * FA, n0 = tn * 16u * FB;
    const uint32_t blocks = (a.cols + HCOMM_GFX_MX_BLOCK - 1u) / HCOMM_GFX_MX_BLOCK, chunks = (blocks + CHUNK_BLOCKS - 1u) / CHUNK_BLOCKS;
    uint64_t row_a[FA], row_b[FB]; // rows past the end: the last one once more, its results are not stored
#pragma unroll
    for (int i = 0; i < FA; ++i) row_a[i] = min(m0 + 16u * i + (lane & 15u), a.m - 1u);
#pragma unroll
    for (int i = 0; i < FB; ++i) row_b[i] = min(n0 + 16u * i + (lane & 15u), a.n - 1u);
    f32x4 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t rank = wave / chunks, chunk = wave - rank * chunks;
    while (rank < a.k) {
        const uint32_t first = chunk * CHUNK_BLOCKS + (lane >> 4) * 4u;
        Run ra[FA], rb[FB];
#pragma unroll
        for (int j = 0; j < FB; ++j) rb[j] = load_run(a.b[rank], row_b[j], first, blocks);
#pragma unroll
        for (int i = 0; i < FA; ++i) ra[i] = load_run(a.a[rank], row_a[i], first, blocks);
        if (chunk == chunks - 1u) {
#pragma unroll
            for (int i = 0; i < FA; ++i) cut_run(ra[i], first, a.cols);
        }
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j) {
                acc[i][j] = mfma<0>(ra[i].block[0], rb[j].block[0], acc[i][j], ra[i].scales, rb[j].scales);
                acc[i][j] = mfma<1>(ra[i].block[1], rb[j].block[1], acc[i][j], ra[i].scales, rb[j].scales);
                acc[i][j] = mfma<2>(ra[i].block[2], rb[j].block[2], acc[i][j], ra[i].scales, rb[j].scales);
                acc[i][j] = mfma<3>(ra[i].block[3], rb[j].block[3], acc[i][j], ra[i].scales, rb[j].scales);
            }
        chunk += 4u;
        while (chunk >= chunks) chunk -= chunks, ++rank;
    }
    if (wave != 0u) {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j) part[wave - 1u][i * FB + j][lane] = acc[i][j];
    }
    __syncthreads();
    if (wave == 0u) {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j) {
                f32x4 v = acc[i][j];
#pragma unroll
                for (int w = 0; w < 3; ++w) v += part[w][i * FB + j][lane];
                const uint32_t col = n0 + 16u * j + (lane & 15u);
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) {
                    const uint32_t row = m0 + 16u * i + (lane >> 4) * 4u + e;
                    if (row < a.m && col < a.n) put(a.dst, a.dtype, row * a.dst_stride + col, v[e]);
                }
            }
    }
}

} // namespace

extern "C" {

int hg_launch_mx_product(void* stream, const void* args)
{
    const HgMxProduct* a = (const HgMxProduct*)args;
    OnDeviceOf device((hipStream_t)stream);
    if (device.err != hipSuccess) return HCCL_E_RUNTIME;
    const dim3 g(a->wgs), b(256);
    switch (a->form) {
        case HG_PRODUCT_DIRECT_16: hipLaunchKernelGGL((k_mx_product_direct<1, 1>), g, b, 0, (hipStream_t)stream, *a); break;
        case HG_PRODUCT_DIRECT_32: hipLaunchKernelGGL((k_mx_product_direct<2, 2>), g, b, 0, (hipStream_t)stream, *a); break;
        default: return HCCL_E_INTERNAL;
    }
    return rc(hipGetLastError());
}

} // extern "C"
