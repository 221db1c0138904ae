// hg_norm.hip - what follows the fold of a tensor-parallel block, and its gradient.
//
// One pass over memory: the wavefronts that share a row keep it in registers (eight elements a lane and group, 64 lanes a
// wavefront), so k partials and the residual are read once, the sums over the row cross the lanes twice and everything
// in between never leaves the registers.  Bound by memory from a few hundred rows on; a single row is bound by the latency of
// its load, two reductions and store.
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

// N sums over the at most 16 wavefronts of a row, the same in all of them: lane w of every 16 fetches wavefront w's.  `box`
// holds N floats for each wavefront of the workgroup and is not written again before every wavefront has passed another
// barrier.
template <uint32_t N> __device__ __forceinline__ void row_sum(float (&v)[N], float* box, uint32_t waves)
{
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if (waves == 1u) return;
    const uint32_t wave = threadIdx.x >> 6, first = wave & ~(waves - 1u), w = threadIdx.x & 15u; // the host makes `waves` a power of two
    if ((threadIdx.x & 63u) == 0u) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) box[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) v[i] = sum16(w < waves ? box[(first + w) * N + i] : 0.0f);
}

__device__ __forceinline__ float inverse_rms(float squares, uint64_t cols, float eps) { return 1.0f / sqrtf(squares / (float)cols + eps); }

#define MAX_WAVES 16u

// ---- forward --------------------------------------------------------------------------------------------------------

// The arguments as the kernel takes them: the runtime copies them at every launch, so few ranks mean few pointers.
template <uint32_t N> struct NormArgs {
    HcommGfxReduceNormDesc d;
    const void* src[N];
    uint32_t waves, rows_per_wg;
};

// DT: type of the matrices, PT: of the parameters, V: groups of eight elements a lane holds, ONE: a workgroup has one row
// (then where it begins is a scalar), TAIL: rows end inside a group, NT: larger than the L2s, so that what is read once and
// what is written passes by them (8,192 x 4,096 of eight ranks 153 -> 138 us; rows off 16-byte boundaries share lines, which
// has to be fetched again then), N: most ranks
template <int DT, int PT, uint32_t V, bool ONE, bool TAIL, bool NT, uint32_t N> __global__ __launch_bounds__(1024) void k_norm(const NormArgs<N> a)
{
    __shared__ float box[2][MAX_WAVES];
    constexpr uint32_t ES = ElemSize<DT>::v, PS = ElemSize<PT>::v, AHEAD = (DT == DT_F32 ? 4u : 8u) / V;
    const uint32_t span = a.waves * 64u, local = ONE ? 0u : threadIdx.x / span, t = threadIdx.x - local * span;
    const uint64_t row = ONE ? blockIdx.x : (uint64_t)blockIdx.x * a.rows_per_wg + local;
    const uint64_t cols = ONE || row < a.d.rows ? a.d.cols : 0u; // a row that is not there has no columns
    const bool tiny = a.d.cols < 8u;
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
        row_sum(s, box[0], a.waves);
        const float r = inverse_rms(s[0], a.d.cols, a.d.eps);
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
        row_sum(s, box[1], a.waves);
        const float r = inverse_rms(s[0], a.d.cols, a.d.eps);
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
template <int DT, int PT, uint32_t V, uint32_t MOST, bool TAIL, bool NT> __global__ __launch_bounds__(MOST) void k_norm_grad(const HgNormGrad a)
{
    __shared__ float box_a[MAX_WAVES * 3], box_b[MAX_WAVES];
    constexpr uint32_t ES = ElemSize<DT>::v, PS = ElemSize<PT>::v;
    const uint32_t span = a.waves * 64u, t = threadIdx.x;
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
    struct Row {
        Raw8<DT> s[V], y[V], dy[V], dz[V];
    };
    auto ask = [&](Row& x, uint32_t r) {
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            const uint32_t at = (v * span + t) * 8u;
            x.s[v] = ask8<DT, TAIL, NT>((const uint8_t*)a.d.sum + r * a.d.sumStride * ES, at, cols, tiny);
            if (has_pre) {
                x.y[v] = ask8<DT, TAIL, NT>((const uint8_t*)a.d.y + r * a.d.yStride * ES, at, cols, tiny);
                x.dz[v] = ask8<DT, TAIL, NT>((const uint8_t*)a.d.dz + r * a.d.dzStride * ES, at, cols, tiny);
            }
            x.dy[v] = ask8<DT, TAIL, NT>((const uint8_t*)a.d.dy + r * a.d.dyStride * ES, at, cols, tiny);
        }
    };
    Row next;
    if (row < end) ask(next, row);
    Raw8<PT> post[V], pre[V], gate[V];
    float d_post[V][8], d_pre[V][8], d_gate[V][8];
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) {
        if (has_pre) pre[v] = ask8<PT, TAIL, false>(a.d.preWeight, (v * span + t) * 8u, cols, tiny);
        if (has_post) post[v] = ask8<PT, TAIL, false>(a.d.postWeight, (v * span + t) * 8u, cols, tiny);
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) d_post[v][e] = d_pre[v][e] = d_gate[v][e] = 0.0f;
    }
    const float each = 1.0f / (float)cols;
    uint32_t gate_row = 0u, gate_end = 0u; // the row of the gate, and the row at which its next one begins
    if (has_gate && row < end) {
        gate_row = row / (uint32_t)a.d.rowsPerGate;
        gate_end = (gate_row + 1u) * (uint32_t)a.d.rowsPerGate;
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) gate[v] = ask8<PT, TAIL, false>((const uint8_t*)a.d.gate + gate_row * a.d.gateStride * PS, (v * span + t) * 8u, cols, tiny);
    }
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) {
        const uint32_t at = (v * span + t) * 8u;
        if (has_pre) settle8<PT, TAIL>(pre[v], at, cols, tiny);
        if (has_post) settle8<PT, TAIL>(post[v], at, cols, tiny);
        if (has_gate && row < end) settle8<PT, TAIL>(gate[v], at, cols, tiny);
    }
    for (; row < end; ++row) {
        Row x = next;
        if (row + 1u < end) ask(next, row + 1u);
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            const uint32_t at = (v * span + t) * 8u;
            settle8<DT, TAIL>(x.s[v], at, cols, tiny);
            settle8<DT, TAIL>(x.dy[v], at, cols, tiny);
            if (has_pre) settle8<DT, TAIL>(x.y[v], at, cols, tiny), settle8<DT, TAIL>(x.dz[v], at, cols, tiny);
        }
        float q[3] = {0.0f, 0.0f, 0.0f}; // sum^2, y^2, dz preWeight y
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            float s[8];
            widen8<DT>(x.s[v], s);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) q[0] = fmaf(s[e], s[e], q[0]);
            if (has_pre) {
                float y[8], z[8], w[8];
                widen8<DT>(x.y[v], y);
                widen8<DT>(x.dz[v], z);
                widen8<PT>(pre[v], w);
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) q[1] = fmaf(y[e], y[e], q[1]), q[2] = fmaf(z[e] * w[e], y[e], q[2]);
            }
        }
        row_sum(q, box_a, a.waves);
        const float r1 = inverse_rms(q[0], cols, a.d.eps), r2 = has_pre ? inverse_rms(q[1], cols, a.d.eps) : 0.0f;
        const float c2 = r2 * (q[2] * each); // mean of dz preWeight y / rms(y): r2 alone never underflows, its powers do
        float g1[V][8]; // g D postWeight, or g D
        float p[1] = {0.0f};
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            float s[8], d[8];
            widen8<DT>(x.s[v], s);
            widen8<DT>(x.dy[v], d);
            if (has_pre) {
                float y[8], z[8], w[8];
                widen8<DT>(x.y[v], y);
                widen8<DT>(x.dz[v], z);
                widen8<PT>(pre[v], w);
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) {
                    const float n = y[e] * r2;
                    d_pre[v][e] = fmaf(z[e], n, d_pre[v][e]);
                    d[e] = fmaf(r2, fmaf(z[e], w[e], -c2 * n), d[e]);
                }
            }
            if (a.d.dResidual) {
                float o[8];
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) o[e] = a.d.residualScale * d[e];
                store8<DT, TAIL, NT>((uint8_t*)a.d.dResidual + row * a.d.dResidualStride * ES, (v * span + t) * 8u, cols, narrow8<DT>(o));
            }
            float w1[8], g[8];
            if (has_post) widen8<PT>(post[v], w1);
            if (has_gate) widen8<PT>(gate[v], g);
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) {
                const float n = has_post ? s[e] * r1 : s[e];
                if (has_gate) {
                    d_gate[v][e] = fmaf(d[e], has_post ? n * w1[e] : n, d_gate[v][e]);
                    d[e] *= g[e];
                }
                if (has_post) {
                    d_post[v][e] = fmaf(d[e], n, d_post[v][e]);
                    d[e] *= w1[e];
                    p[0] = fmaf(d[e], s[e], p[0]);
                }
                g1[v][e] = d[e];
            }
        }
        if (has_post) {
            row_sum(p, box_b, a.waves);
            const float c1 = r1 * (p[0] * each);
#pragma unroll
            for (uint32_t v = 0; v < V; ++v) {
                float s[8];
                widen8<DT>(x.s[v], s);
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) g1[v][e] = r1 * fmaf(-c1, s[e] * r1, g1[v][e]);
            }
        } else if (a.waves > 1u) {
            __syncthreads(); // box_a is free for the next row
        }
#pragma unroll
        for (uint32_t v = 0; v < V; ++v)
            store8<DT, TAIL, NT>((uint8_t*)a.d.dSum + row * a.d.dSumStride * ES, (v * span + t) * 8u, cols, narrow8<DT>(g1[v]));
        if (has_gate && !a.by_gate && (row + 1u == gate_end || row + 1u == end)) { // whole gate rows in one run: theirs are done
            const uint32_t g = gate_row++;
            gate_end += (uint32_t)a.d.rowsPerGate;
#pragma unroll
            for (uint32_t v = 0; v < V; ++v) {
                if (a.d.dGate) store8<PT, TAIL>((uint8_t*)a.d.dGate + g * a.d.dGateStride * PS, (v * span + t) * 8u, cols, narrow8<PT>(d_gate[v]));
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) d_gate[v][e] = 0.0f;
                if (row + 1u < end) {
                    gate[v] = ask8<PT, TAIL, false>((const uint8_t*)a.d.gate + gate_row * a.d.gateStride * PS, (v * span + t) * 8u, cols, tiny);
                    settle8<PT, TAIL>(gate[v], (v * span + t) * 8u, cols, tiny);
                }
            }
        }
    }
    float* mine = (float*)a.d.workspace + (uint64_t)blockIdx.x * a.sums * a.pitch;
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) {
        const uint32_t at = (v * span + t) * 8u; // the workspace's rows hold whole groups
        if (a.at_post >= 0) store8<DT_F32, false>(mine + (uint64_t)a.at_post * a.pitch, at, a.pitch, narrow8<DT_F32>(d_post[v]));
        if (a.at_pre >= 0) store8<DT_F32, false>(mine + (uint64_t)a.at_pre * a.pitch, at, a.pitch, narrow8<DT_F32>(d_pre[v]));
        if (a.at_gate >= 0) store8<DT_F32, false>(mine + (uint64_t)a.at_gate * a.pitch, at, a.pitch, narrow8<DT_F32>(d_gate[v]));
    }
}

// The runs' sums joined, in a fixed order: a workgroup takes 64 columns of one result, four neighbours to a lane, and 64
// of its lanes share a column's runs.
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

template <int DT, int PT, uint32_t V, bool ONE, bool TAIL, bool NT, uint32_t N> int launch_norm_n(hipStream_t st, const HgNorm* a)
{
    NormArgs<N> n;
    n.d = a->d, n.waves = a->waves, n.rows_per_wg = a->rows_per_wg;
    for (uint32_t j = 0; j < N; ++j) n.src[j] = a->src[j];
    hipLaunchKernelGGL((k_norm<DT, PT, V, ONE, TAIL, NT, N>), dim3(a->wgs), dim3(a->waves * 64u * a->rows_per_wg), 0, st, n);
    return rc(hipGetLastError());
}

template <int DT, int PT, uint32_t V, bool ONE> int launch_norm_v(hipStream_t st, const HgNorm* a)
{
    if (a->d.cols % 8u)
        return a->d.k <= 8u ? launch_norm_n<DT, PT, V, ONE, true, false, 8>(st, a) : launch_norm_n<DT, PT, V, ONE, true, false, HCOMM_GFX_MAX_RANKS>(st, a);
    if (a->d.k > 8u) return launch_norm_n<DT, PT, V, ONE, false, true, HCOMM_GFX_MAX_RANKS>(st, a);
    return a->stream ? launch_norm_n<DT, PT, V, ONE, false, true, 8>(st, a) : launch_norm_n<DT, PT, V, ONE, false, false, 8>(st, a);
}

template <int DT, int PT> int launch_norm(hipStream_t st, const HgNorm* a)
{
    if (a->vecs == 2u) return launch_norm_v<DT, PT, 2, true>(st, a);
    return a->rows_per_wg == 1u ? launch_norm_v<DT, PT, 1, true>(st, a) : launch_norm_v<DT, PT, 1, false>(st, a);
}

template <int DT, int PT, bool TAIL, bool NT> int launch_norm_grad_t(hipStream_t st, const HgNormGrad* a)
{
    const dim3 g((uint32_t)a->chunks), b(a->waves * 64u);
    if (a->vecs == 1u) {
        if (a->waves <= 4u) hipLaunchKernelGGL((k_norm_grad<DT, PT, 1, 256, TAIL, NT>), g, b, 0, st, *a);
        else hipLaunchKernelGGL((k_norm_grad<DT, PT, 1, 512, TAIL, NT>), g, b, 0, st, *a);
    } else {
        if (a->waves <= 8u) hipLaunchKernelGGL((k_norm_grad<DT, PT, 2, 512, TAIL, NT>), g, b, 0, st, *a);
        else hipLaunchKernelGGL((k_norm_grad<DT, PT, 2, 1024, TAIL, NT>), g, b, 0, st, *a);
    }
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
    const dim3 g((uint32_t)((a->d.cols + SUM_COLS - 1u) / SUM_COLS), (uint32_t)((a->at_post >= 0) + (a->at_pre >= 0) + (a->at_gate >= 0 ? a->gates : 0u))), b(1024);
    switch (a->d.paramType) {
        case HCOMM_DATA_TYPE_FP16: hipLaunchKernelGGL((k_norm_sums<DT_F16>), g, b, 0, (hipStream_t)stream, *a); break;
        case HCOMM_DATA_TYPE_BFP16: hipLaunchKernelGGL((k_norm_sums<DT_BF16>), g, b, 0, (hipStream_t)stream, *a); break;
        case HCOMM_DATA_TYPE_FP32: hipLaunchKernelGGL((k_norm_sums<DT_F32>), g, b, 0, (hipStream_t)stream, *a); break;
        default: return HCCL_E_PARA;
    }
    return rc(hipGetLastError());
}

} // extern "C"
