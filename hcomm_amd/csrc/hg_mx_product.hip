// hg_mx_product.hip - the product of two matrices in microscaled 4-bit floating point, summed over the ranks that share
// its inner length: dst = sum over r of a[r] * transpose(b[r]).
//
// The matrix instructions take the format as it is stored.  16 x 16 x 128: lane l gives row l % 16 of an operand, block l / 16
// of four neighbours (32 elements, 16 bytes) and that block's scale byte; 32 x 32 x 64: row l % 32, block l / 32 of two.
#include "hg_ops_device.hpp"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef u32x2_raw u32x2;

#define MX_FP4 4 /* element format operand of the matrix instruction */
#define CHUNK_BLOCKS 16u

// acc += a * b under the scales in byte 0
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 acc, uint32_t sa, uint32_t sb)
{
    const i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, MX_FP4, MX_FP4, 0, (int)sa, 0, (int)sb);
}

// the words of a block of which the first n elements count
__device__ __forceinline__ u32x4 kept(uint32_t n)
{
    u32x4 m;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t keep = n > 8u * i ? n - 8u * i : 0u;
        m[i] = keep >= 8u ? 0xffffffffu : (1u << (4u * keep)) - 1u;
    }
    return m;
}

// What a lane holds of one row for one chunk of 16 blocks: of every four neighbours its own (the four lanes of a row read 64
// bytes in one piece then), and the chunk's scales, of which instruction t takes byte lane / 16 of word t.
struct Run {
    u32x4 block[4];
    u32x4 scales;
};

typedef u32x4 __attribute__((aligned(1))) u32x4_at1;
typedef const __attribute__((address_space(1))) uint8_t cg8;

// Blocks [first, first + 16) of a row of `blocks`, 16 at least.  No branch: loads of several runs are to be under way together.
// Past the row's end its last block is read once more, and settle_run, called where the run is used, takes care of it.  g: lane / 16
__device__ __forceinline__ Run load_run(const HgMxView& v, uint32_t row, uint32_t first, uint32_t blocks, uint32_t g)
{
    Run r;
    const uint8_t* p = v.packed + (uint64_t)row * v.packed_stride;
    const uint8_t* s = v.scales + (uint64_t)row * v.scale_stride;
#pragma unroll
    for (uint32_t t = 0; t < 4u; ++t) r.block[t] = ((cgvec*)p)[min(first + 4u * t + g, blocks - 1u)];
    r.scales = *(const __attribute__((address_space(1))) u32x4_at1*)(s + min(first, blocks - CHUNK_BLOCKS));
    return r;
}

// Four blocks from `first` on as the t-th of a run, in rows of fewer than 16; this lane's scale alone in word t.
__device__ __forceinline__ void load_four(Run& r, uint32_t t, const HgMxView& v, uint32_t row, uint32_t first, uint32_t blocks, uint32_t g)
{
    const uint32_t b = min(first + g, blocks - 1u);
    r.block[t] = ((cgvec*)(v.packed + (uint64_t)row * v.packed_stride))[b];
    r.scales[t] = (uint32_t)((cg8*)(v.scales + (uint64_t)row * v.scale_stride))[b];
}

// w shifted down by `by` bytes, 0 from 16 on
__device__ __forceinline__ u32x4 down_by(u32x4 w, uint32_t by)
{
#pragma unroll
    for (uint32_t step = 1; step < 4u; step *= 2u)
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t from = i + step < 4u ? w[i + step < 4u ? i + step : i] : 0u;
            w[i] = (by & (4u * step)) ? from : w[i];
        }
    u32x4 r;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        r[i] = __builtin_amdgcn_alignbit(i < 3u ? w[i < 3u ? i + 1u : i] : 0u, w[i], 8u * (by % 4u));
        r[i] = by < 16u ? r[i] : 0u;
    }
    return r;
}

// A row's last chunk: scales of blocks past the end become 0 (with 2^-127 on both sides the products are far below what
// fp32 holds), elements of the last block past cols become 0.
__device__ __forceinline__ void settle_run(Run& r, uint32_t first, uint32_t blocks, uint32_t cols, uint32_t g)
{
    const uint32_t by = first - min(first, blocks - CHUNK_BLOCKS); // bytes that the fetch went back
    r.scales = down_by(r.scales, by);
    const uint32_t last = blocks - 1u;
    const u32x4 mask = kept(cols - last * HCOMM_GFX_MX_BLOCK);
#pragma unroll
    for (uint32_t t = 0; t < 4u; ++t)
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) r.block[t][i] &= first + 4u * t + g == last ? mask[i] : 0xffffffffu;
}

__device__ __forceinline__ void settle_four(Run& r, uint32_t t, uint32_t first, uint32_t blocks, uint32_t cols, uint32_t g)
{
    const uint32_t last = blocks - 1u;
    const u32x4 mask = kept(cols - last * HCOMM_GFX_MX_BLOCK);
    r.scales[t] = first + g <= last ? r.scales[t] : 0u;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) r.block[t][i] &= first + g == last ? mask[i] : 0xffffffffu;
}

// four neighbours of a row of dst
template <int DT> __device__ __forceinline__ void put4(void* row, uint32_t at, uint32_t n, f32x4 v)
{
    constexpr uint32_t ES = ElemSize<DT>::v;
    uint8_t* p = (uint8_t*)row + (uint64_t)at * ES;
    const float f[8] = {v.x, v.y, v.z, v.w, 0.0f, 0.0f, 0.0f, 0.0f};
    const Raw8<DT> r = narrow8<DT>(f);
    if (at + 4u <= n) {
        if (ES == 4u) *(__attribute__((address_space(1))) u32x4_at4*)p = u32x4{r.w[0], r.w[1], r.w[2 % Raw8<DT>::words], r.w[3 % Raw8<DT>::words]};
        else *(__attribute__((address_space(1))) u32x2_at2*)p = u32x2{r.w[0], r.w[1]};
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e)
            if (at + e < n) st_elem<ES>(p + e * ES, ES == 4u ? r.w[e] : (r.w[e / 2u] >> (16u * (e % 2u))) & 0xffffu);
    }
}

// The arguments as the kernels take them: the runtime copies them at every launch, so few ranks carry few views.
template <uint32_t N> struct ProductArgs {
    HgMxView a[N], b[N];
    void* dst;
    uint64_t dst_stride;
    uint32_t m, n, cols, k;
};

// ---- few rows: the operands go from memory straight into the matrix instructions --------------------------------------
//
// A workgroup owns 16 FA x 16 FB results; its W wavefronts share the inner length (chunk u of all ranks' chunks goes to
// wavefront u % W), each with the next chunk's loads on their way while it multiplies, and add their sums up through LDS in
// a fixed order.
// SHORT: ranks of fewer than 16 blocks.  A chunk holds fours of blocks there, EACH of them: those of one rank, so that the
// ranks spread over the wavefronts, or with a single wavefront the next four of all ranks' fours.
// One row of 8 ranks' 1,024 columns times 8,192 rows: 8.9 us for 35.7 MB (8.5 in a row of such calls), bound by the loads' latency
// and memory.
template <int DT, int FA, int FB, uint32_t W, bool SHORT, uint32_t N> __global__ __launch_bounds__(64 * W) void k_mx_product_direct(const ProductArgs<N> a)
{
    __shared__ f32x4 part[W > 1u ? W : 1u][W > 1u ? FA * FB : 1][W > 1u ? 64 : 1];
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, shift = SHORT ? 0u : 8u * g, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tiles_n = (a.n + 16u * FB - 1u) / (16u * FB);
    const uint32_t tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
    const uint32_t m0 = tm * 16u * FA, n0 = tn * 16u * FB;
    const uint32_t blocks = (a.cols + HCOMM_GFX_MX_BLOCK - 1u) / HCOMM_GFX_MX_BLOCK, chunks = (blocks + CHUNK_BLOCKS - 1u) / CHUNK_BLOCKS;
    const uint32_t fours = (blocks + 3u) / 4u, each = W > 1u ? fours : 4u;
    uint32_t row_a[FA], row_b[FB]; // rows past the end: the last one once more, its results are not stored
#pragma unroll
    for (int i = 0; i < FA; ++i) row_a[i] = min(m0 + 16u * i + (lane & 15u), a.m - 1u);
#pragma unroll
    for (int i = 0; i < FB; ++i) row_b[i] = min(n0 + 16u * i + (lane & 15u), a.n - 1u);
    f32x4 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    struct Chunk {
        Run a[FA], b[FB];
        uint32_t first, rank; // block of its rank
    } c0, c1;
    uint32_t rank = wave / chunks, chunk = wave - rank * chunks; // of the next loads; SHORT: the chunk is a four of blocks
    auto ask = [&](Chunk& c) {
        const uint32_t first = chunk * CHUNK_BLOCKS;
        c.first = first, c.rank = rank;
#pragma unroll
        for (int j = 0; j < FB; ++j) c.b[j] = load_run(a.b[rank], row_b[j], first, blocks, g);
#pragma unroll
        for (int i = 0; i < FA; ++i) c.a[i] = load_run(a.a[rank], row_a[i], first, blocks, g);
        chunk += W;
        while (chunk >= chunks) chunk -= chunks, ++rank;
    };
    auto ask_fours = [&](Chunk& c) {
        c.first = 4u * chunk, c.rank = rank;
#pragma unroll
        for (uint32_t t = 0; t < 4u; ++t) {
            if (t >= each || rank >= a.k) break;
#pragma unroll
            for (int j = 0; j < FB; ++j) load_four(c.b[j], t, a.b[rank], row_b[j], 4u * chunk, blocks, g);
#pragma unroll
            for (int i = 0; i < FA; ++i) load_four(c.a[i], t, a.a[rank], row_a[i], 4u * chunk, blocks, g);
            if (++chunk == fours) chunk = 0u, ++rank;
        }
        if (W > 1u) rank += W - 1u;
    };
    auto multiply_one = [&](Chunk& c, uint32_t t) {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j)
                acc[i][j] = mfma(c.b[j].block[t], c.a[i].block[t], acc[i][j], c.b[j].scales[t] >> shift, c.a[i].scales[t] >> shift);
    };
    auto multiply = [&](Chunk& c) {
        if (SHORT) {
#pragma unroll
            for (uint32_t t = 0; t < 4u; ++t) {
                if (t >= each || c.rank >= a.k) break;
#pragma unroll
                for (int i = 0; i < FA; ++i) settle_four(c.a[i], t, c.first, blocks, a.cols, g);
#pragma unroll
                for (int j = 0; j < FB; ++j) settle_four(c.b[j], t, c.first, blocks, a.cols, g);
                multiply_one(c, t);
                c.first += 4u;
                if (c.first >= blocks) c.first = 0u, ++c.rank;
            }
            return;
        }
        if (c.first + CHUNK_BLOCKS >= blocks) {
#pragma unroll
            for (int i = 0; i < FA; ++i) settle_run(c.a[i], c.first, blocks, a.cols, g);
#pragma unroll
            for (int j = 0; j < FB; ++j) settle_run(c.b[j], c.first, blocks, a.cols, g);
        }
#pragma unroll
        for (uint32_t t = 0; t < 4u; ++t) multiply_one(c, t);
    };
    auto next = [&](Chunk& c) {
        if (SHORT) ask_fours(c);
        else ask(c);
    };
    if (rank < a.k) {
        next(c0);
        for (;;) {
            const bool more1 = rank < a.k;
            if (more1) next(c1);
            multiply(c0);
            if (!more1) break;
            const bool more0 = rank < a.k;
            if (more0) next(c0);
            multiply(c1);
            if (!more0) break;
        }
    }
    if (W > 1u) {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j) part[wave][i * FB + j][lane] = acc[i][j];
        __syncthreads();
    }
    // a lane holds four neighbours of a row of dst
#pragma unroll
    for (uint32_t f = 0; f < FA * FB; ++f)
        if (f % W == wave) {
            f32x4 v = W > 1u ? part[0][f][lane] : acc[f / FB][f % FB];
#pragma unroll
            for (uint32_t w = 1; w < W; ++w) {
                const f32x4 x = part[w][f][lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += x[e];
            }
            const uint32_t row = m0 + 16u * (f / FB) + (lane & 15u), col = n0 + 16u * (f % FB) + (lane >> 4) * 4u;
            if (row < a.m) put4<DT>((uint8_t*)a.dst + row * a.dst_stride * ElemSize<DT>::v, col, a.n, v);
        }
}

// ---- many rows: tiles through LDS ---------------------------------------------------------------------------------------
//
// A workgroup of four wavefronts owns 256 x 256 results, each wavefront 128 x 128 of them in accumulators (16 matrix
// instructions of 32 x 32 x 64 for every 64 columns).  A stage of 256 columns of both operands (64 KiB) is copied to LDS
// without passing through registers while the stage before it is multiplied.  Rows lie in LDS as eight blocks, block b of
// row r at place b ^ (r % 8), so that both the copies (eight whole rows an instruction) and the reads (one block of 32
// rows) meet every bank evenly.  Scales are fetched by one lane a row, eight bytes a stage, and go through LDS too: fetched by
// the lanes that need them, each would touch 32 lines for a quarter of the lanes' worth of new bytes.
// The wavefronts meet once a stage, before its last quarter is multiplied: by then everything of the stage is in
// registers, its buffer takes the stage after the next, and the fragments of the next one arrive behind that quarter.
// 4,096 x 8,192 results of 8 x 1,024 columns: 139 to 142 us, 3.9 PFLOP/s.  The matrix instructions alone, on random operands
// (which hold the clock down) in a loop, reach 6.0 PFLOP/s: 91 us.  The matrix units are busy 51 % of the time; what is left is the
// wait for the copies of 64 KiB a stage, once a stage.

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint64_t u64_at1 __attribute__((aligned(1)));
typedef __attribute__((address_space(3))) uint8_t lds_byte;
typedef __attribute__((address_space(3))) u32x4 lds_vec;
typedef __attribute__((address_space(3))) uint64_t lds_u64;

#define STAGE_BLOCKS 8u
#define TILE_ROWS 256u

template <int T> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 acc, uint32_t sa, uint32_t sb)
{
    const i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc, MX_FP4, MX_FP4, T, (int)sa, T, (int)sb);
}

// One operand's rows of the tile.  Copies go through a buffer descriptor that ends with the matrix' last block: rows
// past it are not read, whatever lies in their place has no result that is stored.  Scales are read by address, those
// of rows past the end from the last row once more.
struct Side {
    uint32_t rows_at[8]; // this wavefront's eight copies of a stage, as distances of their first rows (scalars)
    uint32_t lane_at;    // and from there this lane's row
    uint32_t scale_at;   // distance of the scale row that this lane fetches
    uint32_t bytes;      // of the tile's rows of the matrix
};

__device__ __forceinline__ Side place_side(const HgMxView& v, uint32_t row0, uint32_t rows, uint32_t blocks, uint32_t wave, uint32_t lane)
{
    Side s;
    const uint32_t last = min(rows - row0, TILE_ROWS) - 1u, stride = (uint32_t)v.packed_stride;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) s.rows_at[i] = (wave * 8u + i) * 8u * stride;
    s.lane_at = (lane >> 3) * stride;
    s.scale_at = min(threadIdx.x, last) * (uint32_t)v.scale_stride;
    s.bytes = last * stride + blocks * HCOMM_GFX_MX_BLOCK_BYTES;
    return s;
}

// The stage that begins at block `first` on its way to LDS.  Past the rows' last block that block is copied once more;
// its scale is 0 (fetch_scales), and with 2^-127 on both sides the products are far below what fp32 holds.
__device__ __forceinline__ void copy_stage(lds_byte* to, const Side& s, const HgMxView& v, uint32_t row0, uint32_t wave, uint32_t lane,
                                           uint32_t first, uint32_t blocks)
{
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(v.packed + (uint64_t)row0 * v.packed_stride, 0, (int)s.bytes, HG_BUFFER_WORD3);
    const uint32_t at = s.lane_at + min(first + ((lane & 7u) ^ (lane >> 3)), blocks - 1u) * HCOMM_GFX_MX_BLOCK_BYTES;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(to + (wave * 8u + i) * 1024u), 16,
                                                 (int)(at + s.rows_at[i]), 0, 0, 0);
}

// the eight scales of this lane's row; the host takes this form from STAGE_BLOCKS blocks on
__device__ __forceinline__ uint64_t fetch_scales(const Side& s, const HgMxView& v, uint32_t row0, uint32_t first, uint32_t blocks)
{
    const uint8_t* base = v.scales + (uint64_t)row0 * v.scale_stride + min(first, blocks - STAGE_BLOCKS);
    return *(const __attribute__((address_space(1))) u64_at1*)(base + s.scale_at);
}

// Elements of the last block past cols do not count: one operand's become 0, in the rows that this wavefront has copied.
// n: the elements of it that count, 32 in stages that end with a whole block (a branch around this would end the basic
// block in which the compiler places the matrix instructions).
__device__ __forceinline__ void cut_rows(lds_byte* la, uint32_t block, uint32_t n)
{
    lds_vec* p = (lds_vec*)(la + threadIdx.x * 128u + ((block ^ (threadIdx.x & 7u)) << 4));
    *p = *p & kept(n);
}

// what a wavefront multiplies: four fragments of 32 rows and 64 columns of each operand
struct Fragments {
    u32x4 a[4], b[4];
};

__device__ __forceinline__ void read_fragments(Fragments& f, lds_byte* la, lds_byte* lb, uint32_t at, uint32_t t)
{
    // at: row lane % 32 at place (lane / 32) ^ (row % 8); two blocks on with every t
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) f.a[i] = *(lds_vec*)(la + (at ^ (t << 5)) + i * 4096u);
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) f.b[i] = *(lds_vec*)(lb + (at ^ (t << 5)) + i * 4096u);
}

// a stage's scales of those fragments' rows, shifted so that instruction t takes byte 2 (t % 2) of word t / 2
struct Scales {
    uint64_t a[4], b[4];
};

__device__ __forceinline__ void read_scales(Scales& s, lds_u64* sa, lds_u64* sb, uint32_t lane)
{
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) s.a[i] = sa[i * 32u + (lane & 31u)], s.b[i] = sb[i * 32u + (lane & 31u)];
}

// T: the instruction of the stage; I0 .. I1: which fragments of a
template <uint32_t T, uint32_t I0, uint32_t I1>
__device__ __forceinline__ void multiply(f32x16 (&acc)[4][4], const Fragments& f, const Scales& s, uint32_t shift)
{
    uint32_t xa[4], xb[4];
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i)
        xa[i] = (uint32_t)(s.a[i] >> (32u * (T / 2u))) >> shift, xb[i] = (uint32_t)(s.b[i] >> (32u * (T / 2u))) >> shift;
#pragma unroll
    for (uint32_t i = I0; i < I1; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) acc[i][j] = mfma32<2u * (T % 2u)>(f.b[j], f.a[i], acc[i][j], xb[j], xa[i]);
}

// The compiler's order of what it may move: N times a matrix instruction followed by one read of LDS, by one access to
// memory.  A wavefront issues in order and is alone on its SIMD, so whatever is not placed behind a matrix instruction that
// is still running leaves the matrix unit idle.
template <int N> __device__ __forceinline__ void behind_each(bool reads, bool loads)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (reads) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        if (loads) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
    }
}

// The results of a wavefront, 32 F x 32 F of them from (m0, n0) on, to dst.  Four neighbours of a row lie in a lane; by way of
// LDS (32 KiB of the wavefront's own) they become runs of a row that a store instruction writes in one piece.  All copies have
// arrived and all wavefronts are done with what they read when this begins.
template <int DT, uint32_t F>
__device__ __forceinline__ void store_results(const f32x16 (&acc)[F][F], lds_byte* mine, uint32_t lane, void* dst, uint64_t dst_stride,
                                              uint32_t m0, uint32_t n0, uint32_t rows, uint32_t cols)
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    constexpr uint32_t ES = ElemSize<DT>::v, EDGE = 32u * F, PASS = EDGE * EDGE * ES > 32768u ? F / 2u : F; // fragments of rows at a time
    constexpr uint32_t ROW = EDGE * ES, SWAP = (ROW / 16u < 32u ? ROW / 16u : 32u) - 1u; // bytes of a row; its chunks of 16 change places by row
    constexpr uint32_t LANES = EDGE / 8u;                                                // that read a row
#pragma unroll
    for (uint32_t i0 = 0; i0 < F; i0 += PASS) {
#pragma unroll
        for (uint32_t i = 0; i < PASS; ++i)
#pragma unroll
            for (uint32_t j = 0; j < F; ++j)
#pragma unroll
                for (uint32_t q = 0; q < 4u; ++q) {
                    const f32x16& v = acc[i0 + i][j];
                    const uint32_t row = i * 32u + (lane & 31u), col = j * 32u + 8u * q + 4u * (lane >> 5); // of four results
                    lds_byte* p = mine + row * ROW + (((col * ES / 16u) ^ (row & SWAP)) << 4) + col * ES % 16u;
                    if (ES == 4u) *(lds_vec*)p = u32x4{f32_bits(v[4 * q]), f32_bits(v[4 * q + 1]), f32_bits(v[4 * q + 2]), f32_bits(v[4 * q + 3])};
                    else {
                        const float f[8] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3], 0.0f, 0.0f, 0.0f, 0.0f};
                        const Raw8<DT> r = narrow8<DT>(f);
                        *(lds_u64*)p = (uint64_t)r.w[1] << 32 | r.w[0];
                    }
                }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (uint32_t t = 0; t < PASS * 32u * LANES / 64u; ++t) {
            const uint32_t row = t * (64u / LANES) + lane / LANES, col = (lane % LANES) * 8u;
            Raw8<DT> r;
#pragma unroll
            for (uint32_t h = 0; h < Raw8<DT>::words / 4u; ++h) {
                const u32x4 v = *(lds_vec*)(mine + row * ROW + (((col * ES / 16u + h) ^ (row & SWAP)) << 4));
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) r.w[4u * h + e] = v[e];
            }
            const uint32_t m = m0 + i0 * 32u + row;
            // from the wavefront's first column on: a row may be longer than 2^32 bytes
            if (m < rows && n0 < cols) store8<DT>((uint8_t*)dst + (m * dst_stride + n0) * ES, col, cols - n0, r);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// TAIL: rows end inside a block
template <int DT, bool TAIL, uint32_t N> __global__ __launch_bounds__(256) void k_mx_product_tile(const ProductArgs<N> a)
{
    // four arrays, not one: the compiler then sees that the copies into one pair do not touch the pair that is read
    __shared__ __align__(1024) uint8_t a0[32768], b0[32768], a1[32768], b1[32768];
    __shared__ uint64_t scales[2][2][TILE_ROWS];
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
    const Side ra = place_side(a.a[0], m0, a.m, blocks, wave, lane), rb = place_side(a.b[0], n0, a.n, blocks, wave, lane);
    const uint32_t at = (lane & 31u) * 128u + (((lane >> 5) ^ (lane & 7u)) << 4), shift = 8u * (lane >> 5);
    const uint32_t total = a.k * stages, tail = a.cols % HCOMM_GFX_MX_BLOCK;
    uint32_t rank = 0, stage = 0;       // of the copies and fetches
    uint32_t left = stages, done = 0;   // of the stages that have arrived: how many to the rank's end, how many in all
    uint64_t fetched_a, fetched_b;
    Fragments f0, f1;
    Scales s;
    // where the next stage is: the rank's matrices, read ahead of their use
    HgMxView va = a.a[0], vb = a.b[0];
    // copies and fetches of the next stage; behind the last one that stage once more, which will not count
#define ASK(TO_A, TO_B)                                                                                               \
    {                                                                                                                 \
        copy_stage((lds_byte*)(TO_A), ra, va, m0, wave, lane, stage * STAGE_BLOCKS, blocks);                          \
        copy_stage((lds_byte*)(TO_B), rb, vb, n0, wave, lane, stage * STAGE_BLOCKS, blocks);                          \
        fetched_a = fetch_scales(ra, va, m0, stage * STAGE_BLOCKS, blocks);                                           \
        fetched_b = fetch_scales(rb, vb, n0, stage * STAGE_BLOCKS, blocks);                                           \
        const bool ends = stage + 1u == stages, last = ends && rank + 1u == a.k;                                      \
        stage = last ? stage : ends ? 0u : stage + 1u;                                                                \
        rank = ends && !last ? rank + 1u : rank;                                                                      \
        va = a.a[rank], vb = a.b[rank];                                                                               \
    }
    // what was asked for last has arrived: its scales (and the cut) on their way to LDS ...
#define ARRIVE(LA, S)                                                                                                 \
    {                                                                                                                 \
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                                                              \
        left = left == 0u ? stages - 1u : left - 1u;                                                                  \
        /* scales past the rows' last block are shifted out: the fetch went back by as many */                        \
        const uint32_t out = left == 0u ? (stages * STAGE_BLOCKS - blocks) * 8u : 0u;                                 \
        const uint64_t counts = done++ < total ? ~0ull : 0ull;                                                        \
        scales[S][0][threadIdx.x] = (fetched_a >> out) & counts;                                                      \
        scales[S][1][threadIdx.x] = (fetched_b >> out) & counts;                                                      \
        if (TAIL) cut_rows((lds_byte*)(LA), (blocks - 1u) % STAGE_BLOCKS, left == 0u ? tail : HCOMM_GFX_MX_BLOCK);    \
    }
    // ... and all wavefronts have come this far
#define MEET()                                                                                                        \
    {                                                                                                                 \
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                                                            \
        __builtin_amdgcn_s_barrier();                                                                                 \
        asm volatile("" ::: "memory");                                                                                \
    }
#define FRAGMENTS(F, LA, LB, T) read_fragments(F, (lds_byte*)(LA) + wm * 16384u, (lds_byte*)(LB) + wn * 16384u, at, T);
#define SCALES(S) read_scales(s, (lds_u64*)scales[S][0] + wm * 128u, (lds_u64*)scales[S][1] + wn * 128u, lane);
#define STAGE(LA, LB, NEXT_A, NEXT_B, NEXT)                                                                           \
    {                                                                                                                 \
        FRAGMENTS(f1, LA, LB, 1)                                                                                      \
        multiply<0, 0, 4>(acc, f0, s, shift);                                                                         \
        behind_each<8>(true, false);                                                                                  \
        __builtin_amdgcn_sched_barrier(0);                                                                            \
        FRAGMENTS(f0, LA, LB, 2)                                                                                      \
        multiply<1, 0, 4>(acc, f1, s, shift);                                                                         \
        behind_each<8>(true, false);                                                                                  \
        __builtin_amdgcn_sched_barrier(0);                                                                            \
        FRAGMENTS(f1, LA, LB, 3)                                                                                      \
        multiply<2, 0, 2>(acc, f0, s, shift);                                                                         \
        behind_each<8>(true, false);                                                                                  \
        __builtin_amdgcn_sched_barrier(0);                                                                            \
        ARRIVE(NEXT_A, NEXT)                                                                                          \
        multiply<2, 2, 4>(acc, f0, s, shift);                                                                         \
        __builtin_amdgcn_sched_barrier(0);                                                                            \
        MEET()                                                                                                        \
        Scales now = s;                                                                                               \
        FRAGMENTS(f0, NEXT_A, NEXT_B, 0)                                                                              \
        SCALES(NEXT)                                                                                                  \
        ASK(LA, LB)                                                                                                   \
        multiply<3, 0, 4>(acc, f1, now, shift);                                                                       \
        behind_each<16>(true, true);                                                                                  \
        __builtin_amdgcn_sched_barrier(0);                                                                            \
    }
    ASK(a0, b0)
    ARRIVE(a0, 0)
    MEET()
    ASK(a1, b1)
    FRAGMENTS(f0, a0, b0, 0)
    SCALES(0)
    // stages in pairs, so that which buffers a stage lies in is known to the compiler
#pragma unroll 1
    for (uint32_t pairs = (total + 1u) >> 1; pairs != 0u; --pairs) {
        STAGE(a0, b0, a1, b1, 1)
        STAGE(a1, b1, a0, b0, 0)
    }
    lds_byte* mine = (lds_byte*)(wave == 0u ? a0 : wave == 1u ? b0 : wave == 2u ? a1 : b1);
    store_results<DT, 4>(acc, mine, lane, a.dst, a.dst_stride, m0 + wm * 128u, n0 + wn * 128u, a.m, a.n);
}

// ---- fewer rows: smaller tiles, more stages under way -------------------------------------------------------------------
//
// 64 F x 64 F results to a workgroup, 32 F x 32 F to a wavefront, stages of 32 KiB.  Such launches are bound by how fast a CU
// gets its operands, so of four buffers three are filled while the fourth is multiplied.

template <int DT, uint32_t F, bool TAIL, uint32_t N> __global__ __launch_bounds__(256) void k_mx_product_mid(const ProductArgs<N> a)
{
    // an array to a stage: the compiler then sees that the copies into one do not touch the one that is read
    __shared__ __align__(1024) uint8_t s0[32768], s1[32768], s2[32768], s3[32768];
    __shared__ __align__(16) uint8_t scales[4][2][1024];
    constexpr uint32_t ROWS = 64u * F, LONG = 16u / F, ROW = LONG * HCOMM_GFX_MX_BLOCK_BYTES; // rows of a tile; blocks and bytes of a row of a stage
    constexpr uint32_t HALF = 16384u;                                                        // of a buffer: a's rows, then b's
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1u;
    const uint32_t tiles_n = (a.n + ROWS - 1u) / ROWS;
    const uint32_t tile = block_id(8u), tm = tile / tiles_n, tn = tile - tm * tiles_n, m0 = tm * ROWS, n0 = tn * ROWS;
    const uint32_t blocks = (a.cols + HCOMM_GFX_MX_BLOCK - 1u) / HCOMM_GFX_MX_BLOCK, total = a.k * ((blocks + LONG - 1u) / LONG);
    f32x16 acc[F][F];
#pragma unroll
    for (uint32_t i = 0; i < F; ++i)
#pragma unroll
        for (uint32_t j = 0; j < F; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    // the ranks' matrices have the same strides (the host sees to it)
    const uint32_t last_a = min(a.m - m0, ROWS) - 1u, last_b = min(a.n - n0, ROWS) - 1u;
    const uint32_t stride_a = (uint32_t)a.a[0].packed_stride, stride_b = (uint32_t)a.b[0].packed_stride;
    // what this lane copies in each of its wavefront's four copies of a side: place lane % LONG of row lane / LONG behind the copy's first
    const uint32_t copy_row = wave * 4u * (4u * F) + lane / LONG, place = lane % LONG;
    // and the eight scales that it fetches: the first two wavefronts of a's rows, the others of b's
    const uint32_t half = wave >> 1, scale_row = (threadIdx.x & 127u) / (LONG / 8u), scale_part = (threadIdx.x & 127u) % (LONG / 8u) * 8u;
    const uint32_t scale_at = min(scale_row, half ? last_b : last_a) * (uint32_t)(half ? a.b[0].scale_stride : a.a[0].scale_stride);
    struct Stage {
        uint64_t fetched;
        uint32_t back, first; // how many scales the fetch went back; the stage's first block
    } q0, q1, q2, q3;
    auto copy = [&](lds_byte* to, const HgMxView& v, uint32_t row0, uint32_t last, uint32_t stride, uint32_t first) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            v.packed + (uint64_t)row0 * v.packed_stride, 0, (int)(last * stride + blocks * HCOMM_GFX_MX_BLOCK_BYTES), HG_BUFFER_WORD3);
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t row = copy_row + i * 4u * F, block = min(first + ((place & ~7u) | ((place ^ row) & 7u)), blocks - 1u);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(to + (wave * 4u + i) * 1024u), 16,
                                                     (int)(row * stride + block * HCOMM_GFX_MX_BLOCK_BYTES), 0, 0, 0);
        }
    };
    // of the next stage to ask for; behind the last one that stage again and again, so that what is under way can be counted
    uint32_t rank = 0, first = 0;
    auto ask = [&](lds_byte* to, Stage& q) {
        const HgMxView &va = a.a[rank], &vb = a.b[rank];
        copy(to, va, m0, last_a, stride_a, first);
        copy(to + HALF, vb, n0, last_b, stride_b, first);
        const uint32_t want = first + scale_part, from = min(want, blocks - 8u); // the host takes this form from 8 blocks on
        const uint8_t* s = half ? vb.scales + (uint64_t)n0 * vb.scale_stride : va.scales + (uint64_t)m0 * va.scale_stride;
        q.fetched = *(const __attribute__((address_space(1))) u64_at1*)(s + from + scale_at);
        q.back = want - from;
        q.first = first;
        const bool ends = first + LONG >= blocks, more = rank + 1u < a.k;
        first = ends ? (more ? 0u : first) : first + LONG;
        rank = ends && more ? rank + 1u : rank;
    };
    // The oldest stage asked for has arrived: what is under way is at most the two stages asked for after it, nine loads each.
    uint32_t done = 0;
    auto meet = [&](lds_byte* in, uint32_t set, const Stage& q) {
        asm volatile("s_waitcnt vmcnt(18)" ::: "memory");
        if (TAIL && lane < 16u * F) {
            // elements of the last block past cols do not count: they become 0 in the rows of a that this wavefront has copied
            const uint32_t last = blocks - 1u - q.first, row = wave * 16u * F + lane; // last: the block in its stage, if it is there
            const uint32_t n = last < LONG ? a.cols - (blocks - 1u) * HCOMM_GFX_MX_BLOCK : HCOMM_GFX_MX_BLOCK, at = last < LONG ? last : 0u;
            lds_vec* p = (lds_vec*)(in + row * ROW + ((at & ~7u) | ((at ^ row) & 7u)) * HCOMM_GFX_MX_BLOCK_BYTES);
            *p = *p & kept(n);
        }
        // scales past the rows' last block become 0, on both sides: the products are far below what fp32 holds
        *(lds_u64*)(lds_byte*)&scales[set][half][scale_row * LONG + scale_part] = q.back < 8u ? q.fetched >> (8u * q.back) : 0u;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        ++done;
    };
    const uint32_t r = lane & 31u, g = lane >> 5;
    auto multiply = [&](lds_byte* from, uint32_t set) {
#pragma unroll
        for (uint32_t q = 0; q < LONG / 8u; ++q) {
            uint64_t sa[F], sb[F];
#pragma unroll
            for (uint32_t i = 0; i < F; ++i) {
                sa[i] = *(lds_u64*)(lds_byte*)&scales[set][0][(wm * 32u * F + i * 32u + r) * LONG + q * 8u];
                sb[i] = *(lds_u64*)(lds_byte*)&scales[set][1][(wn * 32u * F + i * 32u + r) * LONG + q * 8u];
            }
#pragma unroll
            for (uint32_t t = 0; t < 4u; ++t) {
                const uint32_t at = r * ROW + (q * 8u + ((2u * t + g) ^ (r & 7u))) * 16u;
                u32x4 x[F], y[F];
#pragma unroll
                for (uint32_t i = 0; i < F; ++i) {
                    x[i] = *(lds_vec*)(from + (wm * 32u * F + i * 32u) * ROW + at);
                    y[i] = *(lds_vec*)(from + HALF + (wn * 32u * F + i * 32u) * ROW + at);
                }
#pragma unroll
                for (uint32_t i = 0; i < F; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < F; ++j)
                        acc[i][j] = mfma32<0>(y[j], x[i], acc[i][j], (uint32_t)(sb[j] >> (16u * t + 8u * g)), (uint32_t)(sa[i] >> (16u * t + 8u * g)));
            }
        }
    };
    ask((lds_byte*)s0, q0);
    ask((lds_byte*)s1, q1);
    ask((lds_byte*)s2, q2);
    // the buffer of the stage before, which all wavefronts are done with when they have met, takes the third stage from here
#pragma unroll 1
    for (;;) {
        meet((lds_byte*)s0, 0, q0);
        ask((lds_byte*)s3, q3);
        multiply((lds_byte*)s0, 0);
        if (done == total) break;
        meet((lds_byte*)s1, 1, q1);
        ask((lds_byte*)s0, q0);
        multiply((lds_byte*)s1, 1);
        if (done == total) break;
        meet((lds_byte*)s2, 2, q2);
        ask((lds_byte*)s1, q1);
        multiply((lds_byte*)s2, 2);
        if (done == total) break;
        meet((lds_byte*)s3, 3, q3);
        ask((lds_byte*)s2, q2);
        multiply((lds_byte*)s3, 3);
        if (done == total) break;
    }
    lds_byte* mine = (lds_byte*)(wave == 0u ? s0 : wave == 1u ? s1 : wave == 2u ? s2 : s3);
    store_results<DT, F>(acc, mine, lane, a.dst, a.dst_stride, m0 + wm * 32u * F, n0 + wn * 32u * F, a.m, a.n);
}

template <int DT, bool SHORT, uint32_t N> int launch(hipStream_t st, const HgMxProduct* a)
{
    ProductArgs<N> p;
    for (uint32_t j = 0; j < N; ++j) p.a[j] = a->a[j], p.b[j] = a->b[j];
    p.dst = a->dst, p.dst_stride = a->dst_stride, p.m = a->m, p.n = a->n, p.cols = a->cols, p.k = a->k;
    const dim3 g(a->wgs);
    switch (a->form) {
        case HG_PRODUCT_DIRECT_16: hipLaunchKernelGGL((k_mx_product_direct<DT, 1, 1, 8, SHORT, N>), g, dim3(512), 0, st, p); break;
        case HG_PRODUCT_DIRECT_32: hipLaunchKernelGGL((k_mx_product_direct<DT, 2, 2, 8, SHORT, N>), g, dim3(512), 0, st, p); break;
        case HG_PRODUCT_WAVE_32: // of short rows alone
            if (!SHORT) return HCCL_E_INTERNAL;
            hipLaunchKernelGGL((k_mx_product_direct<DT, 2, 2, 1, true, N>), g, dim3(64), 0, st, p);
            break;
        case HG_PRODUCT_MID_64:
            if (a->cols % HCOMM_GFX_MX_BLOCK) hipLaunchKernelGGL((k_mx_product_mid<DT, 1, true, N>), g, dim3(256), 0, st, p);
            else hipLaunchKernelGGL((k_mx_product_mid<DT, 1, false, N>), g, dim3(256), 0, st, p);
            break;
        case HG_PRODUCT_MID_128:
            if (a->cols % HCOMM_GFX_MX_BLOCK) hipLaunchKernelGGL((k_mx_product_mid<DT, 2, true, N>), g, dim3(256), 0, st, p);
            else hipLaunchKernelGGL((k_mx_product_mid<DT, 2, false, N>), g, dim3(256), 0, st, p);
            break;
        case HG_PRODUCT_TILE:
            if (a->cols % HCOMM_GFX_MX_BLOCK) hipLaunchKernelGGL((k_mx_product_tile<DT, true, N>), g, dim3(256), 0, st, p);
            else hipLaunchKernelGGL((k_mx_product_tile<DT, false, N>), g, dim3(256), 0, st, p);
            break;
        default: return HCCL_E_INTERNAL;
    }
    return rc(hipGetLastError());
}

template <int DT, uint32_t N> int launch_length(hipStream_t st, const HgMxProduct* a)
{
    return a->cols <= HCOMM_GFX_MX_BLOCK * (CHUNK_BLOCKS - 1u) ? launch<DT, true, N>(st, a) : launch<DT, false, N>(st, a);
}

template <int DT> int launch_ranks(hipStream_t st, const HgMxProduct* a)
{
    if (a->k == 1u) return launch_length<DT, 1>(st, a);
    return a->k <= 8u ? launch_length<DT, 8>(st, a) : launch_length<DT, HCOMM_GFX_MAX_RANKS>(st, a);
}

} // namespace

extern "C" {

int hg_launch_mx_product(void* stream, const void* args)
{
    const HgMxProduct* a = (const HgMxProduct*)args;
    OnDeviceOf device((hipStream_t)stream);
    if (device.err != hipSuccess) return HCCL_E_RUNTIME;
    switch (a->dtype) {
        case DT_F16: return launch_ranks<DT_F16>((hipStream_t)stream, a);
        case DT_BF16: return launch_ranks<DT_BF16>((hipStream_t)stream, a);
        case DT_F32: return launch_ranks<DT_F32>((hipStream_t)stream, a);
        default: return HCCL_E_PARA;
    }
}

} // extern "C"
