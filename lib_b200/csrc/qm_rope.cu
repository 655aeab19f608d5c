// qm_rope.cu — per head RMSNorm with gain and rotary positions of the q and k heads of q|k|v rows in one pass, and its
// backward pass, for sm_100a.
//
//   n = x / sqrt(mean(x^2) + eps), z = n * gain, and each pair (p, q) of z turned by the token's angle:
//   (p cos - q sin, q cos + p sin), angle_i = position * theta^(-2i/rot) / factor_i.
//   Backward, dy the gradient of the result: dz = dy turned back, dgain = sum over tokens and heads of dz * n,
//   dx = r * (dz * gain - n * mean(dz * gain * n)), r = 1 / sqrt(mean(x^2) + eps).
//
// Nothing is read twice and nothing is written that is not a result, so both are bound by memory for a batch of tokens and
// by launch latency for one. A warp takes `chunk` heads of one token: the angles are computed once for all of them, up to
// four heads are in flight at a time, and a head lies in the warp's registers between its load and its store. A lane owns
// V neighbouring pairs per slot; with V = 2 every access is 8 bytes wide (4 for bf16) and a warp's accesses are contiguous,
// in the half-split as in the adjacent order. V = 1 serves what is not aligned for that.
//
// The angle of a far position has lost its fraction in 32 bits (position 10^6 is 0.06 off), so the turns (angle / 2 pi) are
// a float64 product; their fractional part, at most a half, is exact in float64 and loses 2^-25 of a turn in float32.
#include <cuda_bf16.h>
#include <stdint.h>

#include "qm_kernel_args.h"

namespace {

constexpr int HEADS = 4;      // heads in flight of a forward warp
constexpr int BWD_HEADS = 2;  // of a backward warp, which holds two values per element
constexpr int WARPS = 8;

__device__ __forceinline__ void wait_for_inputs() {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Where the V pairs of a slot lie in a head: elements [at, at + V) and [to, to + V). Turning pairs of the half-split order
// are (at + v, to + v); in the adjacent order, and for what does not turn, two vectors side by side hold them.
struct Place {
    int at, to;
    bool there, turns;
};

template <int V>
__device__ __forceinline__ Place place(const QmQkArgs &a, int pair) {
    Place p;
    p.there = pair < a.dim / 2;
    const int half = a.rot / 2;
    p.turns = pair < half;
    if (p.turns && !a.interleaved) {
        p.at = pair;
        p.to = pair + half;
    } else {
        p.at = 2 * pair;
        p.to = 2 * pair + V;
    }
    return p;
}

template <int V>
__device__ __forceinline__ void load_f32(const float *p, float (&v)[V]) {
    if constexpr (V == 2) {
        const float2 t = *reinterpret_cast<const float2 *>(p);
        v[0] = t.x;
        v[1] = t.y;
    } else {
        v[0] = *p;
    }
}

template <int V>
__device__ __forceinline__ void load_any(const void *base, int64_t at, bool bf16, float (&v)[V]) {
    if (!bf16) {
        load_f32<V>(reinterpret_cast<const float *>(base) + at, v);
    } else if constexpr (V == 2) {
        const uint32_t t = *reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint16_t *>(base) + at);
        v[0] = __uint_as_float(t << 16);
        v[1] = __uint_as_float(t & 0xFFFF0000u);
    } else {
        v[0] = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(base)[at] << 16);
    }
}

template <int V>
__device__ __forceinline__ void store_any(void *base, int64_t at, bool bf16, const float (&v)[V]) {
    if (!bf16) {
        float *p = reinterpret_cast<float *>(base) + at;
        if constexpr (V == 2) *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
        else *p = v[0];
    } else {
        __nv_bfloat16 *p = reinterpret_cast<__nv_bfloat16 *>(base) + at;
        if constexpr (V == 2) *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(v[0], v[1]);
        else *p = __float2bfloat16_rn(v[0]);
    }
}

// Turns the pairs of one slot; the angle's cosine and sine are those of pair v.
template <int V>
__device__ __forceinline__ void turn(float (&f)[V], float (&g)[V], const float (&c)[V], const float (&s)[V], bool split) {
    if (split || V == 1) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float p = f[v], q = g[v];
            f[v] = p * c[v] - q * s[v];
            g[v] = q * c[v] + p * s[v];
        }
    } else if constexpr (V == 2) {
        const float p = f[0], q = f[1], r = g[0], t = g[1];
        f[0] = p * c[0] - q * s[0];
        f[1] = q * c[0] + p * s[0];
        g[0] = r * c[1] - t * s[1];
        g[1] = t * c[1] + r * s[1];
    }
}

template <int V, int NP>
struct Lane {
    Place at[NP];
    float cs[NP][V], sn[NP][V];
    bool split;

    __device__ __forceinline__ void places(const QmQkArgs &a, int lane) {
        split = !a.interleaved;
#pragma unroll
        for (int i = 0; i < NP; i++) at[i] = place<V>(a, (i * 32 + lane) * V);
    }
    __device__ __forceinline__ void angles(const QmQkArgs &a, int lane, int token) {
        const double pos = (double)a.pos[token];
#pragma unroll
        for (int i = 0; i < NP; i++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                const int pair = (i * 32 + lane) * V + v;
                cs[i][v] = 1.f;
                sn[i][v] = 0.f;
                if (pair < a.rot / 2) {
                    const double turns = pos * a.freq[pair];
                    sincospif(2.f * (float)(turns - rint(turns)), &sn[i][v], &cs[i][v]);
                }
            }
    }
};

template <int V, int NP>
__device__ __forceinline__ void forward(const QmQkArgs &a) {
    wait_for_inputs();
    const int lane = threadIdx.x & 31;
    const int64_t task = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (task >= (int64_t)a.tokens * a.chunks) return;
    const int token = (int)(task / a.chunks), first = (int)(task % a.chunks) * a.chunk;
    const int last = min(first + a.chunk, a.hq + a.hk);
    const float *row = a.x + (int64_t)token * a.ldx;
    Lane<V, NP> l;
    l.places(a, lane);
    float f[HEADS][NP][V], g[HEADS][NP][V];
    auto fetch = [&](int h0) {
#pragma unroll
        for (int u = 0; u < HEADS; u++)
#pragma unroll
            for (int i = 0; i < NP; i++) {
#pragma unroll
                for (int v = 0; v < V; v++) f[u][i][v] = g[u][i][v] = 0.f;
                if (h0 + u < last && l.at[i].there) {
                    load_f32<V>(row + (int64_t)(h0 + u) * a.dim + l.at[i].at, f[u][i]);
                    load_f32<V>(row + (int64_t)(h0 + u) * a.dim + l.at[i].to, g[u][i]);
                }
            }
    };
    fetch(first);
    l.angles(a, lane, token);
    for (int h0 = first; h0 < last; h0 += HEADS) {
        if (h0 != first) fetch(h0);
#pragma unroll
        for (int u = 0; u < HEADS; u++) {
            const int h = h0 + u;
            if (h >= last) break;
            float r = 1.f;
            if (a.norm) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < NP; i++)
#pragma unroll
                    for (int v = 0; v < V; v++) ss += f[u][i][v] * f[u][i][v] + g[u][i][v] * g[u][i][v];
                r = 1.f / sqrtf(warp_sum(ss) / (float)a.dim + a.eps);
            }
            const bool is_q = h < a.hq;
            const float *gain = is_q ? a.gain_q : a.gain_k;
            void *out = is_q ? a.q : a.k;
            const int64_t base = is_q ? (int64_t)token * a.ldq + (int64_t)h * a.dim : (int64_t)token * a.ldk + (int64_t)(h - a.hq) * a.dim;
#pragma unroll
            for (int i = 0; i < NP; i++) {
                if (!l.at[i].there) continue;
                if (a.norm) {
                    float w[V], z[V];
#pragma unroll
                    for (int v = 0; v < V; v++) w[v] = z[v] = 1.f;
                    if (gain) {
                        load_f32<V>(gain + l.at[i].at, w);
                        load_f32<V>(gain + l.at[i].to, z);
                    }
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        f[u][i][v] *= r * w[v];
                        g[u][i][v] *= r * z[v];
                    }
                }
                if (l.at[i].turns) turn<V>(f[u][i], g[u][i], l.cs[i], l.sn[i], l.split);
                store_any<V>(out, base + l.at[i].at, a.bf16 != 0, f[u][i]);
                store_any<V>(out, base + l.at[i].to, a.bf16 != 0, g[u][i]);
            }
        }
    }
}

// A warp walks tokens; what it adds up for the gains stays in its registers, the CTA's warps are added in warp order and
// qm_qk_gain_sum adds the CTAs in their order: the same bits in every run.
template <int V, int NP>
__device__ __forceinline__ void backward(const QmQkArgs &a) {
    wait_for_inputs();
    extern __shared__ float sums[];   // [WARPS][2][dim] with the gains' gradients
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Lane<V, NP> l;
    l.places(a, lane);
    float df[2][NP][V], dg[2][NP][V];
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < NP; i++)
#pragma unroll
            for (int v = 0; v < V; v++) df[k][i][v] = dg[k][i][v] = 0.f;
    const int64_t tasks = (int64_t)a.tokens * a.chunks;
    for (int64_t task = (int64_t)blockIdx.x * WARPS + warp; task < tasks; task += (int64_t)gridDim.x * WARPS) {
        const int token = (int)(task / a.chunks), first = (int)(task % a.chunks) * a.chunk;
        const int last = min(first + a.chunk, a.hq + a.hk);
        const float *row = a.x + (int64_t)token * a.ldx;
        float *drow = a.dx + (int64_t)token * a.lddx;
        l.angles(a, lane, token);
#pragma unroll
        for (int i = 0; i < NP; i++)
#pragma unroll
            for (int v = 0; v < V; v++) l.sn[i][v] = -l.sn[i][v];   // turned back
        for (int h0 = first; h0 < last; h0 += BWD_HEADS) {
            float f[BWD_HEADS][NP][V], g[BWD_HEADS][NP][V], p[BWD_HEADS][NP][V], q[BWD_HEADS][NP][V];
#pragma unroll
            for (int u = 0; u < BWD_HEADS; u++)
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    const int h = h0 + u;
#pragma unroll
                    for (int v = 0; v < V; v++) f[u][i][v] = g[u][i][v] = p[u][i][v] = q[u][i][v] = 0.f;
                    if (h < last && l.at[i].there) {
                        const bool is_q = h < a.hq;
                        const void *dy = is_q ? a.q : a.k;
                        const int64_t base = is_q ? (int64_t)token * a.ldq + (int64_t)h * a.dim : (int64_t)token * a.ldk + (int64_t)(h - a.hq) * a.dim;
                        if (a.norm) {
                            load_f32<V>(row + (int64_t)h * a.dim + l.at[i].at, f[u][i]);
                            load_f32<V>(row + (int64_t)h * a.dim + l.at[i].to, g[u][i]);
                        }
                        load_any<V>(dy, base + l.at[i].at, a.bf16 != 0, p[u][i]);
                        load_any<V>(dy, base + l.at[i].to, a.bf16 != 0, q[u][i]);
                    }
                }
#pragma unroll
            for (int u = 0; u < BWD_HEADS; u++) {
                const int h = h0 + u;
                if (h >= last) break;
                const bool is_q = h < a.hq;
                const float *gain = is_q ? a.gain_q : a.gain_k;
                float ss = 0.f, dot = 0.f;
                float w[NP][V], z[NP][V];
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    if (l.at[i].turns) turn<V>(p[u][i], q[u][i], l.cs[i], l.sn[i], l.split);
#pragma unroll
                    for (int v = 0; v < V; v++) w[i][v] = z[i][v] = 1.f;
                    if (a.norm && gain && l.at[i].there) {
                        load_f32<V>(gain + l.at[i].at, w[i]);
                        load_f32<V>(gain + l.at[i].to, z[i]);
                    }
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        ss += f[u][i][v] * f[u][i][v] + g[u][i][v] * g[u][i][v];
                        dot += p[u][i][v] * w[i][v] * f[u][i][v] + q[u][i][v] * z[i][v] * g[u][i][v];
                    }
                }
                float r = 1.f, m = 0.f;
                if (a.norm) {
                    ss = warp_sum(ss);
                    dot = warp_sum(dot);
                    r = 1.f / sqrtf(ss / (float)a.dim + a.eps);
                    m = r * dot / (float)a.dim;   // mean of dz * gain * n
                }
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    if (!l.at[i].there) continue;
                    float o[V], t[V];
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        const float nf = f[u][i][v] * r, ng = g[u][i][v] * r;
                        o[v] = r * (p[u][i][v] * w[i][v] - nf * m);
                        t[v] = r * (q[u][i][v] * z[i][v] - ng * m);
                        if (is_q) {
                            df[0][i][v] += p[u][i][v] * nf;
                            dg[0][i][v] += q[u][i][v] * ng;
                        } else {
                            df[1][i][v] += p[u][i][v] * nf;
                            dg[1][i][v] += q[u][i][v] * ng;
                        }
                    }
                    store_any<V>(drow, (int64_t)h * a.dim + l.at[i].at, false, o);
                    store_any<V>(drow, (int64_t)h * a.dim + l.at[i].to, false, t);
                }
            }
        }
    }
    if (!a.partial) return;
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < NP; i++)
            if (l.at[i].there) {
#pragma unroll
                for (int v = 0; v < V; v++) {
                    sums[(warp * 2 + k) * a.dim + l.at[i].at + v] = df[k][i][v];
                    sums[(warp * 2 + k) * a.dim + l.at[i].to + v] = dg[k][i][v];
                }
            }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * a.dim; e += WARPS * 32) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) s += sums[w * 2 * a.dim + e];
        a.partial[(int64_t)blockIdx.x * 2 * a.dim + e] = s;
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_w1(const __grid_constant__ QmQkArgs a) { forward<2, 1>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_w2(const __grid_constant__ QmQkArgs a) { forward<2, 2>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_w4(const __grid_constant__ QmQkArgs a) { forward<2, 4>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_s8(const __grid_constant__ QmQkArgs a) { forward<1, 8>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_grad_w1(const __grid_constant__ QmQkArgs a) { backward<2, 1>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_grad_w2(const __grid_constant__ QmQkArgs a) { backward<2, 2>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_grad_w4(const __grid_constant__ QmQkArgs a) { backward<2, 4>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_grad_s8(const __grid_constant__ QmQkArgs a) { backward<1, 8>(a); }

// One CTA per eight columns of the [2][dim] sums: 32 threads walk the CTAs' rows of a column in float64 (one order, whatever
// the grid), a warp adds its threads.
extern "C" __global__ void __launch_bounds__(256) qm_qk_gain_sum(const __grid_constant__ QmGainSumArgs a) {
    wait_for_inputs();
    const int col = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (col >= 2 * a.dim) return;
    double s = 0.0;
    for (int c = lane; c < a.ctas; c += 32) s += (double)a.partial[(int64_t)c * 2 * a.dim + col];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
        float *out = col < a.dim ? a.dq : a.dk;
        if (out) out[col < a.dim ? col : col - a.dim] = (float)s;
    }
}
