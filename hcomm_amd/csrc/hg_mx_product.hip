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

template <int DT> __device__ __forceinline__ void put(void* dst, uint64_t i, float v)
{
    if (DT == DT_F32) ((__attribute__((address_space(1))) float*)dst)[i] = v;
    else if (DT == DT_BF16) ((__attribute__((address_space(1))) __bf16*)dst)[i] = (__bf16)v;
    else ((__attribute__((address_space(1))) _Float16*)dst)[i] = (_Float16)v;
}

// ---- few rows: the operands go from memory straight into the matrix instructions --------------------------------------
//
// A workgroup owns 16 FA x 16 FB results; its four wavefronts share the inner length (chunk u of all ranks' chunks goes to
// wavefront u % 4) and add their sums up through LDS in a fixed order.
template <int DT, int FA, int FB> __global__ __launch_bounds__(256) void k_mx_product_direct(const HgMxProduct a)
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
                    if (row < a.m && col < a.n) put<DT>(a.dst, row * a.dst_stride + col, v[e]);
                }
            }
    }
}

// ---- many rows: tiles through LDS ---------------------------------------------------------------------------------------
//
// A workgroup of four wavefronts owns 256 x 256 results, each wavefront 128 x 128 of them in accumulators (16 matrix
// instructions of 32 x 32 x 64 for every 64 columns).  A stage of 256 columns of both operands (64 KiB) is copied to LDS
// without passing through registers while the stage before it is multiplied; one barrier a stage tells that all four have
// their copies there and are done with the stage before.  Rows lie in LDS as eight blocks, block b of row r at place b ^ (r % 8),
// so that both the copies (eight whole rows an instruction) and the reads (one block of 32 rows) meet every bank evenly.
// Scales go to registers: eight bytes of a row a stage, of which the two lanes of a row take every other byte.

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint64_t u64_at1 __attribute__((aligned(1)));

#define STAGE_BLOCKS 8u
#define TILE_ROWS 256u

template <int T> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 acc, uint32_t sa, uint32_t sb)
{
    const i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc, MX_FP4, MX_FP4, T, (int)sa, T, (int)sb);
}

typedef __attribute__((address_space(3))) uint8_t lds_byte;
typedef __attribute__((address_space(3))) u32x4 lds_vec;

// one operand's rows of the tile, as distances in bytes: those that this lane copies a block of, those of its four
// fragments' scales; rows past the end are the last one once more, their results are not stored
struct Side {
    uint32_t copy[8], scale[4];
};

__device__ __forceinline__ Side place_side(const HgMxView& v, uint32_t row0, uint32_t rows, uint32_t wave, uint32_t lane, uint32_t frag0)
{
    Side s;
    const uint32_t last = rows - 1u - row0;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) s.copy[i] = min((wave * 8u + i) * 8u + (lane >> 3), last) * (uint32_t)v.packed_stride;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) s.scale[i] = min(frag0 + i * 32u + (lane & 31u), last) * (uint32_t)v.scale_stride;
    return s;
}

// The stage that begins at block `first` on its way to LDS, its scales to registers.  Past the rows' last block that
// block is copied once more and its scale is 0: with 2^-127 on both sides the products are far below what fp32 holds.
__device__ __forceinline__ void stage_side(lds_byte* to, uint64_t (&scale)[4], const Side& s, const HgMxView& v, uint32_t row0, uint32_t wave, uint32_t lane, uint32_t first, uint32_t blocks)
{
    const uint8_t* base = v.packed + (uint64_t)row0 * v.packed_stride;
    const uint32_t block = min(first + ((lane & 7u) ^ (lane >> 3)), blocks - 1u) * HCOMM_GFX_MX_BLOCK_BYTES;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)(base + (s.copy[i] + block)),
                                         (__attribute__((address_space(3))) uint32_t*)(to + (wave * 8u + i) * 1024u), 16, 0, 0);
    const uint32_t from = min(first, blocks - STAGE_BLOCKS); // the host takes this form from STAGE_BLOCKS blocks on
    const uint8_t* scales = v.scales + (uint64_t)row0 * v.scale_stride + from;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) scale[i] = *(const __attribute__((address_space(1))) u64_at1*)(scales + s.scale[i]) >> (8u * (first - from));
}

// elements of the last block past cols do not count: one operand's become 0, a row to a lane
__device__ __forceinline__ void cut_stage(lds_byte* la, uint32_t block, uint32_t n)
{
    lds_vec* p = (lds_vec*)(la + threadIdx.x * 128u + ((block ^ (threadIdx.x & 7u)) << 4));
    u32x4 v = *p;
#pragma unroll
    for (uint32_t q = 0; q < 4u; ++q) {
        const uint32_t keep = n > 8u * q ? n - 8u * q : 0u;
        v[q] &= keep >= 8u ? 0xffffffffu : (1u << (4u * keep)) - 1u;
    }
    *p = v;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ void multiply_stage(f32x16 (&acc)[4][4], lds_byte* la, lds_byte* lb, uint32_t wm, uint32_t wn, uint32_t lane, const uint64_t (&sa)[4], const uint64_t (&sb)[4])
{
    const uint32_t r = lane & 31u, g = lane >> 5;
    uint32_t xa[2][4], xb[2][4]; // this lane's bytes: of instruction t byte 2 (t % 2) of word t / 2
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        xa[0][i] = (uint32_t)sa[i] >> (8u * g), xa[1][i] = (uint32_t)(sa[i] >> 32) >> (8u * g);
        xb[0][i] = (uint32_t)sb[i] >> (8u * g), xb[1][i] = (uint32_t)(sb[i] >> 32) >> (8u * g);
    }
#pragma unroll
    for (uint32_t t = 0; t < 4u; ++t) {
        const uint32_t at = r * 128u + (((2u * t + g) ^ (r & 7u)) << 4);
        u32x4 a[4], b[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            a[i] = *(lds_vec*)(la + (wm * 128u + i * 32u) * 128u + at);
            b[i] = *(lds_vec*)(lb + (wn * 128u + i * 32u) * 128u + at);
        }
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i)
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                if (t % 2u == 0u) acc[i][j] = mfma32<0>(a[i], b[j], acc[i][j], xa[t / 2u][i], xb[t / 2u][j]);
                else acc[i][j] = mfma32<2>(a[i], b[j], acc[i][j], xa[t / 2u][i], xb[t / 2u][j]);
            }
    }
}

// all of this wavefront's copies have arrived; then all wavefronts'
__device__ __forceinline__ void copies_there()
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int DT> __global__ __launch_bounds__(256) void k_mx_product_tile(const HgMxProduct a)
{
    // four arrays, not one: the compiler then sees that the copies into one pair do not touch the pair that is read
    __shared__ __align__(1024) uint8_t a0[32768], b0[32768], a1[32768], b1[32768];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1u;
    const uint32_t tiles_m = (a.m + TILE_ROWS - 1u) / TILE_ROWS, tiles_n = (a.n + TILE_ROWS - 1u) / TILE_ROWS;
    // each XCD walks tiles next to one another, four rows of tiles at a time: its L2 keeps what they share
    const uint32_t tile = block_id(32u), band = tile / (4u * tiles_n), in = tile - band * 4u * tiles_n;
    const uint32_t high = min(4u, tiles_m - band * 4u), tm = band * 4u + in % high, tn = in / high;
    const uint32_t m0 = tm * TILE_ROWS, n0 = tn * TILE_ROWS;
    const uint32_t blocks = (a.cols + HCOMM_GFX_MX_BLOCK - 1u) / HCOMM_GFX_MX_BLOCK, stages = (blocks + STAGE_BLOCKS - 1u) / STAGE_BLOCKS;
    f32x16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    // the ranks' matrices have the same strides (the host sees to it)
    const Side ra = place_side(a.a[0], m0, a.m, wave, lane, wm * 128u), rb = place_side(a.b[0], n0, a.n, wave, lane, wn * 128u);
    uint64_t sa[2][4], sb[2][4];
    uint32_t rank = 0, stage = 0; // of the copies
    const uint32_t total = a.k * stages, tail = a.cols % HCOMM_GFX_MX_BLOCK;
    uint32_t left = stages; // of the products: stages to the rank's end
#define STAGE(TO_A, TO_B, S)                                                                                     \
    {                                                                                                            \
        stage_side((lds_byte*)(TO_A), sa[S], ra, a.a[rank], m0, wave, lane, stage * STAGE_BLOCKS, blocks);       \
        stage_side((lds_byte*)(TO_B), sb[S], rb, a.b[rank], n0, wave, lane, stage * STAGE_BLOCKS, blocks);       \
        if (++stage == stages) stage = 0u, ++rank;                                                               \
    }
#define MULTIPLY(LA, LB, S)                                                                                      \
    {                                                                                                            \
        if (--left == 0u) {                                                                                      \
            left = stages;                                                                                       \
            if (tail) cut_stage((lds_byte*)(LA), (blocks - 1u) % STAGE_BLOCKS, tail);                            \
        }                                                                                                        \
        multiply_stage(acc, (lds_byte*)(LA), (lds_byte*)(LB), wm, wn, lane, sa[S], sb[S]);                       \
    }
    // stages in pairs, so that which buffer a stage lies in is known to the compiler; an odd one goes first
    if (total & 1u) {
        STAGE(a1, b1, 1)
        copies_there();
        if (total > 1u) STAGE(a0, b0, 0)
        MULTIPLY(a1, b1, 1)
    } else {
        STAGE(a0, b0, 0)
    }
#pragma unroll 1
    for (uint32_t pairs = total >> 1; pairs != 0u; --pairs) {
        copies_there();
        STAGE(a1, b1, 1)
        MULTIPLY(a0, b0, 0)
        copies_there();
        if (pairs > 1u) STAGE(a0, b0, 0)
        MULTIPLY(a1, b1, 1)
    }
#undef MULTIPLY
#undef STAGE
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) {
            const uint32_t col = n0 + wn * 128u + j * 32u + (lane & 31u);
#pragma unroll
            for (uint32_t e = 0; e < 16u; ++e) {
                const uint32_t row = m0 + wm * 128u + i * 32u + 8u * (e / 4u) + 4u * (lane >> 5) + e % 4u;
                if (row < a.m && col < a.n) put<DT>(a.dst, row * a.dst_stride + col, acc[i][j][e]);
            }
        }
}

template <int DT> int launch(hipStream_t st, const HgMxProduct* a)
{
    const dim3 g(a->wgs), b(256);
    switch (a->form) {
        case HG_PRODUCT_DIRECT_16: hipLaunchKernelGGL((k_mx_product_direct<DT, 1, 1>), g, b, 0, st, *a); break;
        case HG_PRODUCT_DIRECT_32: hipLaunchKernelGGL((k_mx_product_direct<DT, 2, 2>), g, b, 0, st, *a); break;
        case HG_PRODUCT_TILE: hipLaunchKernelGGL((k_mx_product_tile<DT>), g, b, 0, st, *a); break;
        default: return HCCL_E_INTERNAL;
    }
    return rc(hipGetLastError());
}

} // namespace

extern "C" {

int hg_launch_mx_product(void* stream, const void* args)
{
    const HgMxProduct* a = (const HgMxProduct*)args;
    OnDeviceOf device((hipStream_t)stream);
    if (device.err != hipSuccess) return HCCL_E_RUNTIME;
    switch (a->dtype) {
        case DT_F16: return launch<DT_F16>((hipStream_t)stream, a);
        case DT_BF16: return launch<DT_BF16>((hipStream_t)stream, a);
        case DT_F32: return launch<DT_F32>((hipStream_t)stream, a);
        default: return HCCL_E_PARA;
    }
}

} // extern "C"
