// hg_norm.hip - what follows the fold of a tensor-parallel block, and its gradient.
//
// One pass over memory: the wavefronts that share a row keep it in registers (eight elements a lane and group, 64 lanes a
// wavefront), so k partials and the residual are read once, the sums over the row cross the lanes twice and everything
// in between never leaves the registers.  Bound by memory from a few hundred rows on (medians of the kernels' durations, 8,192 x
// 4,096 bf16 of eight ranks: 138 us for 805 MB, 5.8 TB/s; its gradient: 79 us and 4.6 for the join, 403 MB, 4.8 TB/s); a single row
// is bound by the latency of its load, two reductions and store (5.3 us at 8,192 columns of eight ranks).  Rows that do not begin
// on cache lines take up to half as long again: every access of a wavefront touches a line more, and neighbouring rows share theirs.
#include "hg_ops_device.hpp"

namespace {

// ---- sums over a row ------------------------------------------------------------------------------------------------

template <int CTRL> __device__ __forceinline__ float plus_dpp(float v)
{
    return v + bits_f32((uint32_t)__builtin_amdgcn_mov_dpp((int)f32_bits(v), CTRL, 0xf, 0xf, true));
}

// the sum over 16 neighbouring lanes, in all of them
__device__ __forceinline__ float sum16(float v)
{
    v = plus_dpp<0xB1>(v);     // 1 0 3 2
    v = plus_dpp<0x4E>(v);     // 2 3 0 1
    v = plus_dpp<0x141>(v);    // mirrored in 8
    return plus_dpp<0x140>(v); // mirrored in 16
}

// the sum over the wavefront, in every lane: across its rows of 16 lanes by scalar reads
__device__ __forceinline__ float wave_sum(float v)
{
    const int s = (int)f32_bits(sum16(v));
    const float a = bits_f32((uint32_t)__builtin_amdgcn_readlane(s, 0)), b = bits_f32((uint32_t)__builtin_amdgcn_readlane(s, 16));
    const float c = bits_f32((uint32_t)__builtin_amdgcn_readlane(s, 32)), d = bits_f32((uint32_t)__builtin_amdgcn_readlane(s, 48));
    return (a + b) + (c + d);
}

// What a workgroup has: one row, several of whole wavefronts (1 or 2 each), or several of 1 to 32 lanes.
enum { ONE_ROW, WAVES, LANES };

// N sums over the `span` lanes that share a row, the same in all of them.  Across wavefronts, at most 16: lane w of every 16
// fetches wavefront w's sum from `box`, which holds N floats for each wavefront of the workgroup and is not written again before
// every wavefront has passed another barrier.
template <uint32_t N, int SHARE> __device__ __forceinline__ void row_sum(float (&v)[N], float* box, uint32_t span)
{
    if (SHARE == LANES) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            if (span >= 2u) v[i] = plus_dpp<0xB1>(v[i]);
            if (span >= 4u) v[i] = plus_dpp<0x4E>(v[i]);
            if (span >= 8u) v[i] = plus_dpp<0x141>(v[i]);
            if (span >= 16u) v[i] = plus_dpp<0x140>(v[i]);
            if (span >= 32u) v[i] += __shfl_xor(v[i], 16);
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    const uint32_t waves = span / 64u;
    if (waves == 1u) return;
    const uint32_t wave = threadIdx.x >> 6, first = SHARE == ONE_ROW ? 0u : wave & ~1u, w = threadIdx.x & 15u;
    if ((threadIdx.x & 63u) == 0u) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) box[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) v[i] = sum16(w < waves ? box[(first + w) * N + i] : 0.0f);
}

// 1 / rms of a row from its sum of squares, `each` = 1 / its length.  The instruction is good to one unit in the last place, of
// normal numbers.
__device__ __forceinline__ float inverse_rms(float squares, float each, float eps)
{
    const float m = fmaf(squares, each, eps);
    const bool small = m < 0x1p-100f;
    return __builtin_amdgcn_rsqf(small ? m * 0x1p100f : m) * (small ? 0x1p50f : 1.0f);
}

#define MAX_WAVES 16u

// ---- forward --------------------------------------------------------------------------------------------------------

// The arguments as the kernel takes them: the runtime copies them at every launch, so few ranks mean few pointers.
template <uint32_t N> struct NormArgs {
    HcommGfxReduceNormDesc d;
    const void* src[N];
    uint32_t span, rows_per_wg;
};

// DT: type of the matrices, PT: of the parameters, V: groups of eight elements a lane holds, SHARE: a workgroup has one row
// (where it begins is a scalar then), several of whole wavefronts, or several of fewer lanes, TAIL: rows end inside a group,
// NT: what is read once and what is written passes by the L2s, N: most ranks.
// NT is taken for rows of whole groups that move more than the L2s hold.  8,192 x 4,096 of eight ranks without / with it, us:
// 154 / 139, as a view with a row every 4,099 elements, whose rows share lines, 184 / 174, 4,096 x 8,200: 207 / 203.  More than eight
// ranks take it at any size (with it alone compiled): 16 ranks' 8,192 x 4,096 252 / 216, 1,024 rows 37.5 / 34.5, 64 rows 9.8 / 11,
// a row of 8,192 7.9 / 7.9.  Rows that end inside a group do without: neighbours share lines that would be fetched again.
template <int DT, int PT, uint32_t V, int SHARE, bool TAIL, bool NT, uint32_t N> __global__ __launch_bounds__(1024) void k_norm(const NormArgs<N> a)
{
    __shared__ float box[2][MAX_WAVES];
    constexpr uint32_t ES = ElemSize<DT>::v, PS = ElemSize<PT>::v, AHEAD = (DT == DT_F32 ? 4u : 8u) / V;
    constexpr bool ONE = SHARE == ONE_ROW;
    const uint32_t span = a.span, local = ONE ? 0u : threadIdx.x >> __builtin_ctz(span), t = threadIdx.x - local * span;
    const uint64_t row = ONE ? blockIdx.x : (uint64_t)blockIdx.x * a.rows_per_wg + local;
    const uint64_t cols = ONE || row < a.d.rows ? a.d.cols : 0u; // a row that is not there has no columns
    const bool tiny = a.d.cols < 8u;
    const float each = 1.0f / (float)a.d.cols;
    float f[V][8];
    Raw8<DT> x[AHEAD][V], res[V];
    Raw8<PT> post[V], pre[V], gate[V];
    auto ask = [&](uint32_t j0) {
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j)
            if (j0 + j < a.d.k) {
#pragma unroll
                for (uint32_t v = 0; v < V; ++v)
                    x[j][v] = ask8<DT, TAIL, NT>((const uint8_t*)a.src[j0 + j] + row * a.d.srcStride * ES, (v * span + t) * 8u, cols, tiny);
            }
    };
    auto add = [&](uint32_t j0) {
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j)
            if (j0 + j < a.d.k) {
#pragma unroll
                for (uint32_t v = 0; v < V; ++v) {
                    float g[8];
                    settle8<DT, TAIL>(x[j][v], (v * span + t) * 8u, cols, tiny);
                    widen8<DT>(x[j][v], g);
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e) f[v][e] = j0 + j == 0u ? g[e] : f[v][e] + g[e];
                }
            }
    };
    ask(0);
    // what the row's end needs is asked for before the ranks' sum is waited for
    const uint32_t gate_row = a.d.gate && cols ? (uint32_t)row / (uint32_t)a.d.rowsPerGate : 0u; // the host keeps both below 2^31
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) {
        const uint32_t at = (v * span + t) * 8u;
        if (a.d.residual) res[v] = ask8<DT, TAIL, NT>((const uint8_t*)a.d.residual + row * a.d.residualStride * ES, at, cols, tiny);
        if (a.d.postWeight) post[v] = ask8<PT, TAIL, false>(a.d.postWeight, at, cols, tiny);
        if (a.d.gate) gate[v] = ask8<PT, TAIL, false>((const uint8_t*)a.d.gate + (uint64_t)gate_row * a.d.gateStride * PS, at, cols, tiny);
        if (a.d.preWeight) pre[v] = ask8<PT, TAIL, false>(a.d.preWeight, at, cols, tiny);
    }
    add(0);
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) {
        const uint32_t at = (v * span + t) * 8u;
        if (a.d.residual) settle8<DT, TAIL>(res[v], at, cols, tiny);
        if (a.d.postWeight) settle8<PT, TAIL>(post[v], at, cols, tiny);
        if (a.d.gate) settle8<PT, TAIL>(gate[v], at, cols, tiny);
        if (a.d.preWeight) settle8<PT, TAIL>(pre[v], at, cols, tiny);
    }
    for (uint32_t j0 = AHEAD; j0 < a.d.k; j0 += AHEAD) {
        ask(j0);
        add(j0);
    }
    if (a.d.sum) {
#pragma unroll
        for (uint32_t v = 0; v < V; ++v)
            store8<DT, TAIL, NT>((uint8_t*)a.d.sum + row * a.d.sumStride * ES, (v * span + t) * 8u, cols, narrow8<DT>(f[v]));
    }
    if (a.d.postWeight) {
        float s[1] = {0.0f};
#pragma unroll
        for (uint32_t v = 0; v < V; ++v)
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) s[0] = fmaf(f[v][e], f[v][e], s[0]);
        row_sum<1, SHARE>(s, box[0], span);
        const float r = inverse_rms(s[0], each, a.d.eps);
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            float w[8];
            widen8<PT>(post[v], w);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) f[v][e] = f[v][e] * r * w[e];
        }
    }
    float s[1] = {0.0f};
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) {
        if (a.d.gate) {
            float w[8];
            widen8<PT>(gate[v], w);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) f[v][e] *= w[e];
        }
        if (a.d.residual) {
            float y[8];
            widen8<DT>(res[v], y);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) f[v][e] = fmaf(a.d.residualScale, y[e], f[v][e]);
        }
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) s[0] = fmaf(f[v][e], f[v][e], s[0]);
        store8<DT, TAIL, NT>((uint8_t*)a.d.y + row * a.d.yStride * ES, (v * span + t) * 8u, cols, narrow8<DT>(f[v]));
    }
    if (a.d.preWeight) {
        row_sum<1, SHARE>(s, box[1], span);
        const float r = inverse_rms(s[0], each, a.d.eps);
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            float w[8];
            widen8<PT>(pre[v], w);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) f[v][e] = f[v][e] * r * w[e];
            store8<DT, TAIL, NT>((uint8_t*)a.d.z + row * a.d.zStride * ES, (v * span + t) * 8u, cols, narrow8<DT>(f[v]));
        }
    }
}

// ---- gradient ---------------------------------------------------------------------------------------------------------

// A run of rows to a workgroup: the parameters' gradients stay in registers over the run, and the row after the one at work
// is on its way while the sums of this one cross the lanes.
// SUB: rows of 1 to 32 lanes, several to a wavefront, each taking every so many units of the run's rows (a unit: the rows
// of one row of the gate where its gradient is written at once, else one row); their sums are joined at the run's end.
// LEAN: rows so long that neither the next one nor the parameters have registers beside them: those are asked for again.
// What is not there is taken as what leaves the formulas as they are (a gate of 1, a dz of 0), not by branches around them.
//
// Which of them, for 33.5M elements in bf16, us:
//   SUB up to 256 columns: 96 at 64 columns, 419 with a wavefront to each row (56 of its lanes idle);
//   V = 1 up to 4,096: 82 to 95, 4.9 to 4.2 TB/s of 5.1 that a copy reaches;
//   V = 2 up to 8,192, 8 wavefronts of 256 registers, the second group's sums in LDS: 88 to 93 (fp32 190; 258 with these sums
//   in registers that spill); LEAN with V = 1 and 16 wavefronts: 200;
//   LEAN with V = 2 above: 167 to 170 (fp32 270 to 285); 815 and more with everything held and spilled, 228 to 255 (fp32 335) with
//   rows read again for each of their uses.  Bound by the latency of a row's loads, with one workgroup to a CU.
template <int DT, int PT, uint32_t V, uint32_t MOST, bool SUB, bool LEAN, bool TAIL, bool NT>
__global__ __launch_bounds__(MOST) void k_norm_grad(const HgNormGrad a)
{
    __shared__ float box_a[MAX_WAVES * 3], box_b[MAX_WAVES];
    constexpr uint32_t ES = ElemSize<DT>::v, PS = ElemSize<PT>::v;
    constexpr int SHARE = SUB ? LANES : ONE_ROW;
    constexpr int HT = V == 1u ? DT_F32 : PT; // parameters are held as this
    constexpr bool PASS = NT && !LEAN;
    const uint32_t span = a.span;
    uint32_t t = SUB ? threadIdx.x & (span - 1u) : threadIdx.x;
    const uint64_t cols = a.d.cols;
    const bool tiny = cols < 8u;
    const bool has_post = a.d.postWeight != nullptr, has_pre = a.d.preWeight != nullptr, has_gate = a.d.gate != nullptr;
    uint32_t row, end; // the host keeps rows below 2^31
    if (a.by_gate) {
        const uint32_t per = (uint32_t)a.chunks_per_gate, g = blockIdx.x / per, part = blockIdx.x - g * per;
        const uint32_t begin = g * (uint32_t)a.d.rowsPerGate, stop = min(begin + (uint32_t)a.d.rowsPerGate, (uint32_t)a.d.rows);
        row = min(begin + part * (uint32_t)a.chunk_rows, stop);
        end = min(row + (uint32_t)a.chunk_rows, stop);
    } else {
        row = blockIdx.x * (uint32_t)a.chunk_rows;
        end = min(row + (uint32_t)a.chunk_rows, (uint32_t)a.d.rows);
    }
    const uint32_t sets = 64u >> __builtin_ctz(span), unit = a.unit; // of lanes; rows a set takes before it leaves out the other sets'
    if (SUB) row += (threadIdx.x >> __builtin_ctz(span)) * unit;
    uint32_t unit_end = SUB ? row + unit : 0u;
    auto after = [&](uint32_t r) { return SUB && r + 1u == unit_end ? r + 1u + (sets - 1u) * unit : r + 1u; };
    struct Row {
        Raw8<DT> s, y, dy, dz; // without a norm in front of the next block y and dz stay 0
    };
    constexpr uint32_t HELD = LEAN ? 1u : V; // groups whose parameters are held
    auto ask_one = [&](Raw8<DT>& x, const void* m, uint64_t stride, uint32_t r, uint32_t v) {
        x = ask8<DT, TAIL, PASS>((const uint8_t*)m + r * stride * ES, (v * span + t) * 8u, cols, tiny);
    };
    auto ask = [&](Row& x, uint32_t r, uint32_t v) {
        ask_one(x.s, a.d.sum, a.d.sumStride, r, v);
        if (has_pre) ask_one(x.y, a.d.y, a.d.yStride, r, v), ask_one(x.dz, a.d.dz, a.d.dzStride, r, v);
        else if (LEAN) x.y = x.dz = zeros8<DT>(); // not held from row to row
        ask_one(x.dy, a.d.dy, a.d.dyStride, r, v);
    };
    auto ask_row = [&](Row (&x)[V], uint32_t r) {
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) ask(x[v], r, v);
    };
    auto settle = [&](Raw8<DT>& x, uint32_t v) { settle8<DT, TAIL>(x, (v * span + t) * 8u, cols, tiny); };
    auto settle_row = [&](Row& x, uint32_t v) {
        settle(x.s, v);
        if (has_pre) settle(x.y, v), settle(x.dz, v);
        settle(x.dy, v);
    };
    // A parameter's group in fp32; one that is not there: what leaves the formulas as they are without it.
    auto param = [&](const void* m, uint32_t v, float missing, float (&w)[8]) {
        const float each_is[8] = {missing, missing, missing, missing, missing, missing, missing, missing};
        Raw8<PT> p = narrow8<PT>(each_is);
        if (m) ask8_into<PT, TAIL, false>(p, m, (v * span + t) * 8u, cols, tiny);
        settle8<PT, TAIL>(p, (v * span + t) * 8u, cols, tiny);
        widen8<PT>(p, w);
    };
    auto hold = [&](const void* m, uint32_t v, float missing) {
        float w[8];
        param(m, v, missing, w);
        return narrow8<HT>(w); // exact: fp32, or the type it came in
    };
    auto gate_at = [&](uint32_t r) { return has_gate ? (const uint8_t*)a.d.gate + r * a.d.gateStride * PS : (const uint8_t*)nullptr; };
    // What a lane asks for behind this is not asked for before it: LEAN has room for little at a time.
    auto apart = [] {
        if (LEAN) {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    Row next[V];
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) next[v].y = next[v].dz = zeros8<DT>();
    if (!LEAN && row < end) ask_row(next, row);
    uint32_t gate_row = 0u, gate_end = 0u; // the row of the gate, and the row at which its next one begins
    Raw8<HT> post[HELD], pre[HELD], gate[HELD];
    // a row of the gate that is asked for and not settled, where `fresh`; else it goes to `gate` at once
    Raw8<PT> asked[HT == PT ? 1u : HELD];
    bool fresh = false;
    auto take_gate = [&](uint32_t r) {
        gate_row = r / (uint32_t)a.d.rowsPerGate;
        gate_end = (gate_row + 1u) * (uint32_t)a.d.rowsPerGate;
        if (!LEAN) {
#pragma unroll
            for (uint32_t v = 0; v < HELD; ++v) {
                const uint32_t at = (v * span + t) * 8u;
                if constexpr (HT == PT) gate[v] = ask8<PT, TAIL, false>(gate_at(gate_row), at, cols, tiny);
                else asked[v] = ask8<PT, TAIL, false>(gate_at(gate_row), at, cols, tiny);
            }
            fresh = true;
        }
    };
    if (!LEAN) {
#pragma unroll
        for (uint32_t v = 0; v < HELD; ++v)
            pre[v] = hold(a.d.preWeight, v, 0.0f), post[v] = hold(a.d.postWeight, v, 1.0f), gate[v] = hold(nullptr, v, 1.0f);
    }
    if (has_gate && row < end) take_gate(row);
    float d_post[8], d_pre[8], d_gate[8];
#pragma unroll
    for (uint32_t e = 0; e < 8u; ++e) d_post[e] = d_pre[e] = d_gate[e] = 0.0f;
    // the second group's sums and results stay in LDS
    enum { POST, PRE, GATE, RESULT };
    __shared__ __align__(16) float4 second[V > 1u ? 4 : 1][2][V > 1u ? MOST : 1u];
    auto keep = [&](int which, const float (&d)[8]) {
        second[which][0][t] = make_float4(d[0], d[1], d[2], d[3]);
        second[which][1][t] = make_float4(d[4], d[5], d[6], d[7]);
    };
    auto kept = [&](int which, float (&d)[8]) {
        const float4 l = second[which][0][t], h = second[which][1][t];
        d[0] = l.x, d[1] = l.y, d[2] = l.z, d[3] = l.w, d[4] = h.x, d[5] = h.y, d[6] = h.z, d[7] = h.w;
    };
    if (V > 1u) keep(POST, d_post), keep(PRE, d_pre), keep(GATE, d_gate);
    const float each = 1.0f / (float)cols;
    while (row < end) {
        const uint32_t following = after(row);
        if (LEAN) asm volatile("" : "+v"(t)); // no addresses held from row to row
        Row x[V];
        if (!LEAN) {
#pragma unroll
            for (uint32_t v = 0; v < V; ++v) x[v] = next[v];
            if (following < end) ask_row(next, following);
        } else {
            ask_row(x, row);
        }
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) settle_row(x[v], v);
        float q[3] = {0.0f, 0.0f, 0.0f}; // sum^2, y^2, dz preWeight y
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            Row& h = x[v];
            float s[8], y[8], z[8], w[8];
            widen8<DT>(h.s, s);
            widen8<DT>(h.y, y);
            widen8<DT>(h.dz, z);
            if (LEAN) param(a.d.preWeight, v, 0.0f, w);
            else widen8<HT>(pre[LEAN ? 0u : v], w);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) {
                q[0] = fmaf(s[e], s[e], q[0]);
                q[1] = fmaf(y[e], y[e], q[1]);
                q[2] = fmaf(z[e] * w[e], y[e], q[2]);
            }
        }
        row_sum<3, SHARE>(q, box_a, span);
        const float r1 = has_post ? inverse_rms(q[0], each, a.d.eps) : 1.0f, r2 = has_pre ? inverse_rms(q[1], each, a.d.eps) : 0.0f;
        const float c2 = r2 * (r2 * (q[2] * each)); // mean of dz preWeight y / rms(y), by 1 / rms(y): r2 y never underflows with y
        float p[1] = {0.0f};
        if (!LEAN && fresh) {
#pragma unroll
            for (uint32_t v = 0; v < HELD; ++v) {
                const uint32_t at = (v * span + t) * 8u;
                if constexpr (HT == PT) settle8<PT, TAIL>(gate[v], at, cols, tiny);
                else {
                    float w[8];
                    settle8<PT, TAIL>(asked[v], at, cols, tiny);
                    widen8<PT>(asked[v], w);
                    gate[v] = narrow8<HT>(w);
                }
            }
            fresh = false;
        }
        // adds to the parameters' gradients and to p; n: s / rms(s) or s, o: g D postWeight
        auto group = [&](uint32_t v, float (&to_post)[8], float (&to_pre)[8], float (&to_gate)[8], float (&o)[8]) {
            apart();
            Row& h = x[v];
            float s[8], d[8], y[8], z[8], w[8], g[8];
            widen8<DT>(h.s, s);
            widen8<DT>(h.dy, d);
            widen8<DT>(h.y, y);
            widen8<DT>(h.dz, z);
            if (LEAN) param(a.d.preWeight, v, 0.0f, w);
            else widen8<HT>(pre[LEAN ? 0u : v], w);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) {
                const float n = y[e] * r2;
                to_pre[e] = fmaf(z[e], n, to_pre[e]);
                d[e] = fmaf(-c2, n, fmaf(r2, z[e] * w[e], d[e]));
            }
            if (a.d.dResidual) {
                float res[8];
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) res[e] = a.d.residualScale * d[e];
                store8<DT, TAIL, NT>((uint8_t*)a.d.dResidual + row * a.d.dResidualStride * ES, (v * span + t) * 8u, cols, narrow8<DT>(res));
            }
            if (LEAN) param(a.d.postWeight, v, 1.0f, w), param(gate_at(gate_row), v, 1.0f, g);
            else widen8<HT>(post[LEAN ? 0u : v], w), widen8<HT>(gate[LEAN ? 0u : v], g);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) {
                const float n = s[e] * r1;
                to_gate[e] = fmaf(d[e], n * w[e], to_gate[e]);
                d[e] *= g[e];
                to_post[e] = fmaf(d[e], n, to_post[e]);
                o[e] = d[e] * w[e];
                p[0] = fmaf(o[e], s[e], p[0]);
            }
        };
        float first[8];
        group(0u, d_post, d_pre, d_gate, first);
        if (V > 1u) {
            float post2[8], pre2[8], gate2[8], o[8];
            kept(POST, post2), kept(PRE, pre2), kept(GATE, gate2);
            group(1u, post2, pre2, gate2, o);
            keep(POST, post2), keep(PRE, pre2), keep(GATE, gate2), keep(RESULT, o);
        }
        float c1 = 0.0f;
        if (has_post) {
            row_sum<1, SHARE>(p, box_b, span);
            c1 = r1 * (p[0] * each);
        } else if (span > 64u) {
            __syncthreads(); // box_a is free for the next row
        }
        auto finish = [&](uint32_t v, float (&o)[8]) {
            apart();
            if (has_post) {
                float s[8];
                widen8<DT>(x[v].s, s);
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) o[e] = r1 * fmaf(-c1, s[e] * r1, o[e]);
            }
            store8<DT, TAIL, NT>((uint8_t*)a.d.dSum + row * a.d.dSumStride * ES, (v * span + t) * 8u, cols, narrow8<DT>(o));
        };
        finish(0u, first);
        if (V > 1u) {
            float o[8];
            kept(RESULT, o);
            finish(1u, o);
        }
        if (has_gate && !a.by_gate && (following >= gate_end || following >= end)) {
            if (a.d.dGate) { // whole rows of the gate in one run: this one is done
                uint8_t* to = (uint8_t*)a.d.dGate + gate_row * a.d.dGateStride * PS;
                store8<PT, TAIL>(to, t * 8u, cols, narrow8<PT>(d_gate));
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) d_gate[e] = 0.0f;
                if (V > 1u) {
                    float o[8];
                    kept(GATE, o);
                    store8<PT, TAIL>(to, (span + t) * 8u, cols, narrow8<PT>(o));
                    keep(GATE, d_gate);
                }
            }
            if (following < end) take_gate(following);
        }
        if (SUB && row + 1u == unit_end) unit_end = following + unit;
        row = following;
    }
    // this run's sums; rows that shared a wavefront's lanes are joined first
    float* mine = (float*)a.d.workspace + (uint64_t)blockIdx.x * a.sums * a.pitch;
    auto join = [&](float (&d)[8]) {
        if (SUB) {
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e)
                for (uint32_t far = span; far < 64u; far *= 2u) d[e] += __shfl_xor(d[e], (int)far);
        }
        return !SUB || threadIdx.x < span; // who leaves them
    };
    auto leave = [&](int at, int which, float (&d)[8]) {
        if (at < 0) return;
        // the workspace's rows hold whole groups
        if (join(d)) store8<DT_F32, false>(mine + (uint64_t)at * a.pitch, t * 8u, a.pitch, narrow8<DT_F32>(d));
        if (V > 1u) {
            float o[8];
            kept(which, o);
            store8<DT_F32, false>(mine + (uint64_t)at * a.pitch, (span + t) * 8u, a.pitch, narrow8<DT_F32>(o));
        }
    };
    leave(a.at_post, POST, d_post);
    leave(a.at_pre, PRE, d_pre);
    leave(a.at_gate, GATE, d_gate);
    if (a.by_gate && a.at_gate < 0) { // the run has all rows of its row of the gate
        uint8_t* to = (uint8_t*)a.d.dGate + blockIdx.x * a.d.dGateStride * PS;
        if (join(d_gate)) store8<PT, TAIL>(to, t * 8u, cols, narrow8<PT>(d_gate));
        if (V > 1u) {
            float o[8];
            kept(GATE, o);
            store8<PT, TAIL>(to, (span + t) * 8u, cols, narrow8<PT>(o));
        }
    }
}

// The runs' sums joined, in a fixed order (4.6 to 4.9 us: the latency of a launch and of a chain of loads): a workgroup takes 64
// columns of one result, four neighbours to a lane, and 64 of its lanes share a column's runs.
#define SUM_COLS 64u

template <int PT> __global__ __launch_bounds__(1024) void k_norm_sums(const HgNormGrad a)
{
    __shared__ float part[16][SUM_COLS];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, in = lane & 15u;
    const uint32_t results = (a.at_post >= 0) + (a.at_pre >= 0);
    uint32_t first = 0u, n = (uint32_t)a.chunks, which;
    uint8_t* out;
    if (blockIdx.y < results) {
        const bool post = blockIdx.y == 0u && a.at_post >= 0;
        which = (uint32_t)(post ? a.at_post : a.at_pre);
        out = (uint8_t*)(post ? a.d.dPostWeight : a.d.dPreWeight);
    } else {
        const uint32_t g = blockIdx.y - results;
        which = (uint32_t)a.at_gate;
        first = g * (uint32_t)a.chunks_per_gate;
        n = (uint32_t)a.chunks_per_gate;
        out = (uint8_t*)a.d.dGate + g * a.d.dGateStride * ElemSize<PT>::v;
    }
    const uint64_t step = a.sums * (a.pitch / 4u); // in vectors of four
    cgvec* p = (cgvec*)a.d.workspace + first * step + which * (a.pitch / 4u) + blockIdx.x * (SUM_COLS / 4u) + in;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (uint32_t i = wave * 4u + (lane >> 4); i < n; i += 64u) {
        const u32x4 v = p[i * step];
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) s[e] += bits_f32(v[e]);
    }
#pragma unroll
    for (uint32_t e = 0; e < 4u; ++e) {
        s[e] += __shfl_xor(s[e], 16);
        s[e] += __shfl_xor(s[e], 32);
        if (lane < 16u) part[wave][in * 4u + e] = s[e];
    }
    __syncthreads();
    const uint32_t col = blockIdx.x * SUM_COLS + threadIdx.x;
    if (threadIdx.x < SUM_COLS && col < a.d.cols) {
        float t = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < 16u; ++w) t += part[w][threadIdx.x];
        if (PT == DT_F32) ((float*)out)[col] = t;
        else if (PT == DT_BF16) ((__bf16*)out)[col] = (__bf16)t;
        else ((_Float16*)out)[col] = (_Float16)t;
    }
}

template <int DT, int PT, uint32_t V, int SHARE, bool TAIL, bool NT, uint32_t N> int launch_norm_n(hipStream_t st, const HgNorm* a)
{
    NormArgs<N> n;
    n.d = a->d, n.span = a->span, n.rows_per_wg = a->rows_per_wg;
    for (uint32_t j = 0; j < N; ++j) n.src[j] = a->src[j];
    hipLaunchKernelGGL((k_norm<DT, PT, V, SHARE, TAIL, NT, N>), dim3(a->wgs), dim3(a->span * a->rows_per_wg), 0, st, n);
    return rc(hipGetLastError());
}

template <int DT, int PT, uint32_t V, int SHARE> int launch_norm_v(hipStream_t st, const HgNorm* a)
{
    if (a->d.cols % 8u)
        return a->d.k <= 8u ? launch_norm_n<DT, PT, V, SHARE, true, false, 8>(st, a)
                            : launch_norm_n<DT, PT, V, SHARE, true, false, HCOMM_GFX_MAX_RANKS>(st, a);
    if (a->d.k > 8u) return launch_norm_n<DT, PT, V, SHARE, false, true, HCOMM_GFX_MAX_RANKS>(st, a);
    return a->stream ? launch_norm_n<DT, PT, V, SHARE, false, true, 8>(st, a) : launch_norm_n<DT, PT, V, SHARE, false, false, 8>(st, a);
}

template <int DT, int PT> int launch_norm(hipStream_t st, const HgNorm* a)
{
    if (a->vecs == 2u) return launch_norm_v<DT, PT, 2, ONE_ROW>(st, a);
    if (a->span < 64u) return launch_norm_v<DT, PT, 1, LANES>(st, a);
    return a->rows_per_wg == 1u ? launch_norm_v<DT, PT, 1, ONE_ROW>(st, a) : launch_norm_v<DT, PT, 1, WAVES>(st, a);
}

template <int DT, int PT, bool TAIL, bool NT> int launch_norm_grad_t(hipStream_t st, const HgNormGrad* a)
{
    const dim3 g((uint32_t)a->chunks), b(a->span < 64u ? 64u : a->span);
    if (a->span > 512u) hipLaunchKernelGGL((k_norm_grad<DT, PT, 2, 1024, false, true, TAIL, NT>), g, b, 0, st, *a);
    else if (a->vecs == 2u) hipLaunchKernelGGL((k_norm_grad<DT, PT, 2, 512, false, false, TAIL, NT>), g, b, 0, st, *a);
    else if (a->span >= 64u) hipLaunchKernelGGL((k_norm_grad<DT, PT, 1, 512, false, false, TAIL, NT>), g, b, 0, st, *a);
    else hipLaunchKernelGGL((k_norm_grad<DT, PT, 1, 64, true, false, TAIL, NT>), g, b, 0, st, *a);
    return rc(hipGetLastError());
}

template <int DT, int PT> int launch_norm_grad(hipStream_t st, const HgNormGrad* a)
{
    if (a->d.cols % 8u) return launch_norm_grad_t<DT, PT, true, false>(st, a);
    return a->stream ? launch_norm_grad_t<DT, PT, false, true>(st, a) : launch_norm_grad_t<DT, PT, false, false>(st, a);
}

} // namespace

extern "C" {

int hg_launch_norm(void* stream, const void* args)
{
    const HgNorm* a = (const HgNorm*)args;
    OnDeviceOf device((hipStream_t)stream);
    if (device.err != hipSuccess) return HCCL_E_RUNTIME;
    const hipStream_t st = (hipStream_t)stream;
    const bool wide = a->d.paramType == HCOMM_DATA_TYPE_FP32;
    switch (a->d.dataType) {
        case HCOMM_DATA_TYPE_FP16: return wide ? launch_norm<DT_F16, DT_F32>(st, a) : launch_norm<DT_F16, DT_F16>(st, a);
        case HCOMM_DATA_TYPE_BFP16: return wide ? launch_norm<DT_BF16, DT_F32>(st, a) : launch_norm<DT_BF16, DT_BF16>(st, a);
        case HCOMM_DATA_TYPE_FP32: return launch_norm<DT_F32, DT_F32>(st, a);
        default: return HCCL_E_PARA;
    }
}

int hg_launch_norm_grad(void* stream, const void* args)
{
    const HgNormGrad* a = (const HgNormGrad*)args;
    OnDeviceOf device((hipStream_t)stream);
    if (device.err != hipSuccess) return HCCL_E_RUNTIME;
    const hipStream_t st = (hipStream_t)stream;
    const bool wide = a->d.paramType == HCOMM_DATA_TYPE_FP32;
    switch (a->d.dataType) {
        case HCOMM_DATA_TYPE_FP16: return wide ? launch_norm_grad<DT_F16, DT_F32>(st, a) : launch_norm_grad<DT_F16, DT_F16>(st, a);
        case HCOMM_DATA_TYPE_BFP16: return wide ? launch_norm_grad<DT_BF16, DT_F32>(st, a) : launch_norm_grad<DT_BF16, DT_BF16>(st, a);
        case HCOMM_DATA_TYPE_FP32: return launch_norm_grad<DT_F32, DT_F32>(st, a);
        default: return HCCL_E_PARA;
    }
}

int hg_launch_norm_sums(void* stream, const void* args)
{
    const HgNormGrad* a = (const HgNormGrad*)args;
    OnDeviceOf device((hipStream_t)stream);
    if (device.err != hipSuccess) return HCCL_E_RUNTIME;
    const uint64_t results = (a->at_post >= 0) + (a->at_pre >= 0) + (a->at_gate >= 0 ? a->gates : 0u);
    const dim3 g((uint32_t)((a->d.cols + SUM_COLS - 1u) / SUM_COLS), (uint32_t)results), b(1024);
    switch (a->d.paramType) {
        case HCOMM_DATA_TYPE_FP16: hipLaunchKernelGGL((k_norm_sums<DT_F16>), g, b, 0, (hipStream_t)stream, *a); break;
        case HCOMM_DATA_TYPE_BFP16: hipLaunchKernelGGL((k_norm_sums<DT_BF16>), g, b, 0, (hipStream_t)stream, *a); break;
        case HCOMM_DATA_TYPE_FP32: hipLaunchKernelGGL((k_norm_sums<DT_F32>), g, b, 0, (hipStream_t)stream, *a); break;
        default: return HCCL_E_PARA;
    }
    return rc(hipGetLastError());
}

} // extern "C"
