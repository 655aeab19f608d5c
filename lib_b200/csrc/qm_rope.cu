// qm_rope.cu — per head RMSNorm with gain and rotary positions of the q and k heads of q|k|v rows in one pass, and its
// backward pass, for sm_100a.
//
//   n = x / sqrt(mean(x^2) + eps), z = n * gain, and each pair (p, q) of z turned by the token's angle:
//   (p cos - q sin, q cos + p sin), angle_i = position * theta^(-2i/rot) / factor_i.
//   Backward, dy the gradient of the result: dz = dy turned back, dgain = sum over tokens and heads of dz * n,
//   dx = r * (dz * gain - n * mean(dz * gain * n)), r = 1 / sqrt(mean(x^2) + eps).
//
// Nothing is read twice and nothing is written that is not a result, so both are bound by memory for a batch of tokens and
// by launch latency for one. A warp takes `chunk` query heads (or key heads) of one token: the angles, and with them the
// products of gains, cosines and sines, are computed once for all of them, four heads are in flight at a time and share one
// reduction (each step halves the values a lane holds, so four sums cost nine steps instead of twenty), and a head lies in
// the warp's registers between its load and its store. A lane owns V neighbouring pairs per slot; with V = 2 every access is
// 8 bytes wide (4 for bf16) and a warp's accesses are contiguous, in the half-split as in the adjacent order. V = 1 serves
// what is not aligned for that.
//
// The angle of a far position has lost its fraction in 32 bits (position 10^6 is 0.06 off), so the turns (angle / 2 pi) are
// a product in 64-bit fixed point, position times the fraction of a turn in units of 2^-64, whose overflow is the whole turns:
// what is left, in a few integer instructions, is off by at most 2^-64 of a turn for each position, before it is rounded to
// float32, whose relative error is what the sine of a slow pair's small angle takes over. (Only its upper 32 bits: off by
// 1.5e-4 of itself at position 1 in the last of 64 pairs of theta 500000. The same in float64 kept the FP64 pipe busy:
// 52 -> 45 us at the size below, with a grid that needs no division to find its heads.)
//
// One B200, 40 heads of 128, half-split: 8192 tokens to bf16 44.7 us (5.6 TB/s, 0.86 of the measured copy rate; the first form
// with one reduction per head and gains read for every head 64 us, bound by instruction issue); 4096 tokens backward 49.6 us
// (4.2 TB/s, 0.65; without the gains' gradients 45.9); one token 4.3 us, the cost of a launch.
#include <cuda_bf16.h>
#include <stdint.h>

#include "qm_kernel_args.h"

namespace {

constexpr int HEADS = 4;   // heads in flight of a warp
constexpr int WARPS = 8;

__device__ __forceinline__ void wait_for_inputs() {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The sums over the warp of four values; lane l gets that of value l / 8.
__device__ __forceinline__ float warp_sum4(const float (&s)[4]) {
    const int lane = threadIdx.x & 31;
    const bool high = lane & 16, odd = lane & 8;
    float a = high ? s[2] : s[0], b = high ? s[3] : s[1];
    a += __shfl_xor_sync(0xffffffffu, high ? s[0] : s[2], 16);
    b += __shfl_xor_sync(0xffffffffu, high ? s[1] : s[3], 16);
    float c = odd ? b : a;
    c += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    return c;
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

template <int V, bool BF16>
__device__ __forceinline__ void store_any(void *base, int64_t at, const float (&v)[V]) {
    if constexpr (!BF16) {
        float *p = reinterpret_cast<float *>(base) + at;
        if constexpr (V == 2) *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
        else *p = v[0];
    } else {
        __nv_bfloat16 *p = reinterpret_cast<__nv_bfloat16 *>(base) + at;
        if constexpr (V == 2) *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(v[0], v[1]);
        else *p = __float2bfloat16_rn(v[0]);
    }
}

// In the adjacent order two vectors of two hold (p0, q0), (p1, q1): from there to (p0, p1), (q0, q1), and back.
template <int V>
__device__ __forceinline__ void regroup(float (&f)[V], float (&g)[V], bool adjacent) {
    if constexpr (V == 2) {
        const float t = adjacent ? g[0] : f[1];
        g[0] = adjacent ? f[1] : g[0];
        f[1] = t;
    }
}
// f(p, q, pair) for every pair of a slot, in either order, without moving anything.
template <int V, class F>
__device__ __forceinline__ void pairs(float (&f)[V], float (&g)[V], bool adjacent, F each) {
    if constexpr (V == 1) {
        each(f[0], g[0], 0);
    } else if (adjacent) {
        each(f[0], f[1], 0);
        each(g[0], g[1], 1);
    } else {
        each(f[0], g[0], 0);
        each(f[1], g[1], 1);
    }
}

template <int V, int NP>
struct Lane {
    Place at[NP];
    float cs[NP][V], sn[NP][V];
    float w[NP][V], z[NP][V];   // the gains of the pairs' elements

    __device__ __forceinline__ void places(const QmQkArgs &a, int lane) {
#pragma unroll
        for (int i = 0; i < NP; i++) at[i] = place<V>(a, (i * 32 + lane) * V);
    }
    __device__ __forceinline__ void angles(const QmQkArgs &a, int lane, int token) {
        const uint64_t pos = (uint64_t)(int64_t)a.pos[token];
#pragma unroll
        for (int i = 0; i < NP; i++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                const int pair = (i * 32 + lane) * V + v;
                cs[i][v] = 1.f;
                sn[i][v] = 0.f;
                if (pair < a.rot / 2) {
                    const int64_t turns = (int64_t)(pos * a.freq[pair]);   // of 2^-64 turns, between minus and plus a half
                    sincospif((float)turns * 0x1p-63f, &sn[i][v], &cs[i][v]);
                }
            }
    }
    __device__ __forceinline__ void gains(const QmQkArgs &a, const float *gain) {
#pragma unroll
        for (int i = 0; i < NP; i++) {
#pragma unroll
            for (int v = 0; v < V; v++) w[i][v] = z[i][v] = 1.f;
            if (a.norm && gain && at[i].there) {
                load_f32<V>(gain + at[i].at, w[i]);
                load_f32<V>(gain + at[i].to, z[i]);
                regroup<V>(w[i], z[i], a.interleaved);
            }
        }
    }
};

// A CTA's share: heads [first, last), all of them query heads or all key heads; its warps take tokens.
struct Share {
    int first, last;
    bool is_q;
    __device__ __forceinline__ explicit Share(const QmQkArgs &a) {
        const int c = blockIdx.y;
        is_q = c < a.q_chunks;
        first = is_q ? c * a.chunk : a.hq + (c - a.q_chunks) * a.chunk;
        last = min(first + a.chunk, is_q ? a.hq : a.hq + a.hk);
    }
    // element 0 of the first head in the q or k row of a token
    __device__ __forceinline__ int64_t row(const QmQkArgs &a, int token) const {
        return is_q ? (int64_t)token * a.ldq + (int64_t)first * a.dim : (int64_t)token * a.ldk + (int64_t)(first - a.hq) * a.dim;
    }
};

template <int V, int NP, bool BF16>
__device__ __forceinline__ void forward(const QmQkArgs &a) {
    wait_for_inputs();
    const int lane = threadIdx.x & 31;
    const int token = blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (token >= a.tokens) return;
    const Share t(a);
    const bool adjacent = a.interleaved != 0;
    const float *row = a.x + (int64_t)token * a.ldx + (int64_t)t.first * a.dim;
    Lane<V, NP> l;
    l.places(a, lane);
    float f[HEADS][NP][V], g[HEADS][NP][V];
    auto fetch = [&](int h0) {
        const float *p = row + (h0 - t.first) * a.dim;
#pragma unroll
        for (int u = 0; u < HEADS; u++)
#pragma unroll
            for (int i = 0; i < NP; i++) {
#pragma unroll
                for (int v = 0; v < V; v++) f[u][i][v] = g[u][i][v] = 0.f;
                if (h0 + u < t.last && l.at[i].there) {
                    load_f32<V>(p + u * a.dim + l.at[i].at, f[u][i]);
                    load_f32<V>(p + u * a.dim + l.at[i].to, g[u][i]);
                }
            }
    };
    fetch(t.first);
    l.gains(a, t.is_q ? a.gain_q : a.gain_k);
    l.angles(a, lane, token);
    // (p, q) -> r (p w c - q z s, q z c + p w s)
    float wc[NP][V], zs[NP][V], zc[NP][V], ws[NP][V];
#pragma unroll
    for (int i = 0; i < NP; i++)
#pragma unroll
        for (int v = 0; v < V; v++) {
            wc[i][v] = l.w[i][v] * l.cs[i][v];
            ws[i][v] = l.w[i][v] * l.sn[i][v];
            zc[i][v] = l.z[i][v] * l.cs[i][v];
            zs[i][v] = l.z[i][v] * l.sn[i][v];
        }
    void *out = t.is_q ? a.q : a.k;
    const int64_t base = t.row(a, token);
    for (int h0 = t.first; h0 < t.last; h0 += HEADS) {
        if (h0 != t.first) fetch(h0);
        float r = 1.f;   // lane l: the factor of head l / 8
        if (a.norm) {
            float ss[HEADS];
#pragma unroll
            for (int u = 0; u < HEADS; u++) {
                ss[u] = 0.f;
#pragma unroll
                for (int i = 0; i < NP; i++)
#pragma unroll
                    for (int v = 0; v < V; v++) ss[u] += f[u][i][v] * f[u][i][v] + g[u][i][v] * g[u][i][v];
            }
            r = __frsqrt_rn(warp_sum4(ss) * a.inv_dim + a.eps);
        }
#pragma unroll
        for (int u = 0; u < HEADS; u++) {
            const float ru = __shfl_sync(0xffffffffu, r, 8 * u);
            if (h0 + u >= t.last) break;
            const int64_t at = base + (h0 - t.first + u) * a.dim;
#pragma unroll
            for (int i = 0; i < NP; i++) {
                if (!l.at[i].there) continue;
                if (l.at[i].turns) {
                    pairs<V>(f[u][i], g[u][i], adjacent, [&](float &p, float &q, int v) {
                        const float first = p * wc[i][v] - q * zs[i][v];
                        q = ru * (q * zc[i][v] + p * ws[i][v]);
                        p = ru * first;
                    });
                } else {   // (apart: zero times an infinite neighbour is not zero)
                    pairs<V>(f[u][i], g[u][i], adjacent, [&](float &p, float &q, int v) {
                        p *= ru * wc[i][v];
                        q *= ru * zc[i][v];
                    });
                }
                store_any<V, BF16>(out, at + l.at[i].at, f[u][i]);
                store_any<V, BF16>(out, at + l.at[i].to, g[u][i]);
            }
        }
    }
}

// Two heads as they come from memory; gradients keep their type until they are used.
template <int V, int NP, bool BF16>
struct Pair {
    float f[2][NP][V], g[2][NP][V];
    uint32_t p[2][NP][V], q[2][NP][V];   // float32 bits, or in element 0 the bf16 of the whole vector

    __device__ __forceinline__ static void raw(const void *base, int64_t at, uint32_t (&v)[V]) {
        if constexpr (!BF16) {
            float t[V];
            load_f32<V>(reinterpret_cast<const float *>(base) + at, t);
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = __float_as_uint(t[i]);
        } else if constexpr (V == 2) {
            v[0] = *reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint16_t *>(base) + at);
        } else {
            v[0] = reinterpret_cast<const uint16_t *>(base)[at];
        }
    }
    __device__ __forceinline__ static void values(const uint32_t (&v)[V], float (&t)[V]) {
        if constexpr (!BF16) {
#pragma unroll
            for (int i = 0; i < V; i++) t[i] = __uint_as_float(v[i]);
        } else {
            t[0] = __uint_as_float(v[0] << 16);
            if constexpr (V == 2) t[1] = __uint_as_float(v[0] & 0xFFFF0000u);
        }
    }
};

// A warp walks tokens, two heads at a time, the next two on their way while two are worked on; what it adds up for the gains
// stays in its registers, the CTA's warps are added in warp order and qm_qk_gain_sum adds the CTAs in their order: the same
// bits in every run.
template <int V, int NP, bool BF16>
__device__ __forceinline__ void backward(const QmQkArgs &a) {
    wait_for_inputs();
    extern __shared__ float sums[];   // [WARPS][dim] with the gains' gradients
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Share t(a);
    const bool adjacent = a.interleaved != 0;
    Lane<V, NP> l;
    l.places(a, lane);
    l.gains(a, t.is_q ? a.gain_q : a.gain_k);
    const void *dy = t.is_q ? a.q : a.k;
    float df[NP][V], dg[NP][V];
#pragma unroll
    for (int i = 0; i < NP; i++)
#pragma unroll
        for (int v = 0; v < V; v++) df[i][v] = dg[i][v] = 0.f;
    const int stride = gridDim.x * WARPS;
    auto fetch = [&](Pair<V, NP, BF16> &b, int token, int h0) {
        const float *row = a.x + (int64_t)token * a.ldx + (int64_t)h0 * a.dim;
        const int64_t base = t.row(a, token) + (h0 - t.first) * a.dim;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < NP; i++) {
#pragma unroll
                for (int v = 0; v < V; v++) {
                    b.f[u][i][v] = b.g[u][i][v] = 0.f;
                    b.p[u][i][v] = b.q[u][i][v] = 0u;
                }
                if (h0 + u < t.last && l.at[i].there) {
                    if (a.norm) {
                        load_f32<V>(row + u * a.dim + l.at[i].at, b.f[u][i]);
                        load_f32<V>(row + u * a.dim + l.at[i].to, b.g[u][i]);
                    }
                    b.raw(dy, base + u * a.dim + l.at[i].at, b.p[u][i]);
                    b.raw(dy, base + u * a.dim + l.at[i].to, b.q[u][i]);
                }
            }
    };
    auto work = [&](Pair<V, NP, BF16> &b, int token, int h0) {
        float *drow = a.dx + (int64_t)token * a.lddx + (int64_t)h0 * a.dim;
        if (h0 == t.first) l.angles(a, lane, token);
        float p[2][NP][V], q[2][NP][V], sum[4] = {0.f, 0.f, 0.f, 0.f};   // the squares of both heads, then their products
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < NP; i++) {
                b.values(b.p[u][i], p[u][i]);
                b.values(b.q[u][i], q[u][i]);
                regroup<V>(b.f[u][i], b.g[u][i], adjacent);
                regroup<V>(p[u][i], q[u][i], adjacent);
#pragma unroll
                for (int v = 0; v < V; v++) {
                    if (l.at[i].turns) {   // turned back
                        const float y = p[u][i][v], z = q[u][i][v];
                        p[u][i][v] = y * l.cs[i][v] + z * l.sn[i][v];
                        q[u][i][v] = z * l.cs[i][v] - y * l.sn[i][v];
                    }
                    sum[u] += b.f[u][i][v] * b.f[u][i][v] + b.g[u][i][v] * b.g[u][i][v];
                    sum[2 + u] += p[u][i][v] * b.f[u][i][v] * l.w[i][v] + q[u][i][v] * b.g[u][i][v] * l.z[i][v];
                }
            }
        // dx = r (dz gain - n (r mean(dz gain x))), n = r x: no factor is far from the values themselves, so heads of any
        // magnitude keep their bits as long as their squares fit float32 (r^3, as one factor for x, would overflow below
        // 1e-13 without eps and vanish above 1e13)
        float s = 0.f, r = 1.f;
        if (a.norm) {
            s = warp_sum4(sum) * a.inv_dim;
            r = __frsqrt_rn(s + a.eps);
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const float ru = __shfl_sync(0xffffffffu, r, 8 * u), mu = a.norm ? ru * __shfl_sync(0xffffffffu, s, 16 + 8 * u) : 0.f;
            if (h0 + u >= t.last) break;
#pragma unroll
            for (int i = 0; i < NP; i++) {
                if (!l.at[i].there) continue;
                float o[V], e[V];
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const float x = ru * b.f[u][i][v], y = ru * b.g[u][i][v], c = p[u][i][v], d = q[u][i][v];
                    df[i][v] += c * x;
                    dg[i][v] += d * y;
                    o[v] = ru * (c * l.w[i][v] - x * mu);
                    e[v] = ru * (d * l.z[i][v] - y * mu);
                }
                regroup<V>(o, e, adjacent);
                store_any<V, false>(drow, u * a.dim + l.at[i].at, o);
                store_any<V, false>(drow, u * a.dim + l.at[i].to, e);
            }
        }
    };
    auto after = [&](int &token, int &h0) {
        h0 += 2;
        if (h0 >= t.last) {
            h0 = t.first;
            token += stride;
        }
    };
    int token = blockIdx.x * WARPS + warp, h0 = t.first;
    if constexpr (NP <= 2) {
        Pair<V, NP, BF16> b, c;
        if (token < a.tokens) fetch(b, token, h0);
        while (token < a.tokens) {
            int token2 = token, h2 = h0;
            after(token2, h2);
            if (token2 < a.tokens) fetch(c, token2, h2);
            work(b, token, h0);
            if (token2 >= a.tokens) break;
            token = token2;
            h0 = h2;
            after(token, h0);
            if (token < a.tokens) fetch(b, token, h0);
            work(c, token2, h2);
        }
    } else {   // (two such pairs do not fit in the registers)
        for (; token < a.tokens; after(token, h0)) {
            Pair<V, NP, BF16> b;
            fetch(b, token, h0);
            work(b, token, h0);
        }
    }
    if (!a.partial) return;
#pragma unroll
    for (int i = 0; i < NP; i++)
        if (l.at[i].there) {
            regroup<V>(df[i], dg[i], adjacent);
#pragma unroll
            for (int v = 0; v < V; v++) {
                sums[warp * a.dim + l.at[i].at + v] = df[i][v];
                sums[warp * a.dim + l.at[i].to + v] = dg[i][v];
            }
        }
    __syncthreads();
    for (int e = threadIdx.x; e < a.dim; e += WARPS * 32) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) s += sums[w * a.dim + e];
        a.partial[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.dim + e] = s;
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_w1(const __grid_constant__ QmQkArgs a) { forward<2, 1, false>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_w2(const __grid_constant__ QmQkArgs a) { forward<2, 2, false>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_w4(const __grid_constant__ QmQkArgs a) { forward<2, 4, false>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_s8(const __grid_constant__ QmQkArgs a) { forward<1, 8, false>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_w1_b(const __grid_constant__ QmQkArgs a) { forward<2, 1, true>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_w2_b(const __grid_constant__ QmQkArgs a) { forward<2, 2, true>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_w4_b(const __grid_constant__ QmQkArgs a) { forward<2, 4, true>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_norm_s8_b(const __grid_constant__ QmQkArgs a) { forward<1, 8, true>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32, 3) qm_qk_grad_w1(const __grid_constant__ QmQkArgs a) { backward<2, 1, false>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32, 2) qm_qk_grad_w2(const __grid_constant__ QmQkArgs a) { backward<2, 2, false>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_grad_w4(const __grid_constant__ QmQkArgs a) { backward<2, 4, false>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_grad_s8(const __grid_constant__ QmQkArgs a) { backward<1, 8, false>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32, 3) qm_qk_grad_w1_b(const __grid_constant__ QmQkArgs a) { backward<2, 1, true>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32, 2) qm_qk_grad_w2_b(const __grid_constant__ QmQkArgs a) { backward<2, 2, true>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_grad_w4_b(const __grid_constant__ QmQkArgs a) { backward<2, 4, true>(a); }
extern "C" __global__ void __launch_bounds__(WARPS * 32) qm_qk_grad_s8_b(const __grid_constant__ QmQkArgs a) { backward<1, 8, true>(a); }

// A CTA takes 32 columns of the query (blockIdx.y 0) or key gain, its 32 warps share the CTAs' rows, everything in float64
// and in one order.
extern "C" __global__ void __launch_bounds__(1024) qm_qk_gain_sum(const __grid_constant__ QmGainSumArgs a) {
    wait_for_inputs();
    __shared__ double part[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    const int first = blockIdx.y ? a.q_ctas : 0, last = blockIdx.y ? a.ctas : a.q_ctas;
    double s = 0.0;
    if (col < a.dim) {
#pragma unroll 4
        for (int c = first + warp; c < last; c += 32) s += (double)a.partial[(int64_t)c * a.dim + col];
    }
    part[warp][lane] = s;
    __syncthreads();
    s = part[lane][warp];   // column `warp` of this CTA
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int out_col = blockIdx.x * 32 + warp;
    float *out = blockIdx.y ? a.dk : a.dq;
    if (lane == 0 && out_col < a.dim && out) out[out_col] = (float)s;
}
