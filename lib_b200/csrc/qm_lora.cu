// qm_lora.cu — low-rank adapters of many requests at once beside a shared projection, for sm_100a.
//
//   y[t] = base[t] + s B (A f(x[t])) with the A, B and s of token t's adapter; tokens without one keep their base row.
//   Backward: u = s A x, v = s B^T dy, dx = base + A^T v, dA = sum_t v x^T, dB = sum_t dy u^T over an adapter's tokens.
//
// Everything is a product with a matrix of at most 128 rows, so what bounds it is the wide side: x, base and y, dy, dx.
// Three kinds of products cover both directions, each over tiles of 64 tokens of one adapter:
//   shrink  low[t][r]  = sum_c x[t][c] w[r][c]   (x with A; dy with the transposed B)
//   expand  y[t][c]    = base[t][c] + sum_r low[t][r] w[r][c]
//   outer   grad[r][c] = sum_t low[t][r] x[t][c]
// The 16-bit operands are multiplied as they are. low is a float32 sum; where it is an operand it is taken as the sum of
// three bf16 (8 bits each: all 24 bits of the value), one mma for each, so no rounding to 16 bits enters a result.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "qm_kernel_args.h"
#include "qm_pipe.cuh"

namespace {

using qm::smem_u32;

__device__ __forceinline__ void wait_for_inputs() {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float peer_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 peer_f32x2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
// 16 bytes of which the first `bytes` are read, the others zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t bf_bits(float v) { return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)); }

// v as a sum of three bf16: the next 8 bits of what the ones before leave. An infinity stays in the first.
__device__ __forceinline__ void split3(float v, uint32_t (&p)[3]) {
    p[0] = bf_bits(v);
    const float h = __uint_as_float(p[0] << 16);
    const float rest = isfinite(h) ? v - h : 0.f;
    p[1] = bf_bits(rest);
    p[2] = bf_bits(rest - __uint_as_float(p[1] << 16));
}

struct Tile {
    int slot, first, count;   // slot -1: no adapter
};

// False behind the last tile.
__device__ __forceinline__ bool get_tile(const QmLoraBatchArgs &a, int i, Tile *t) {
    if (a.list) {
        if (i >= a.tiles[0]) return false;
        const int4 w = *reinterpret_cast<const int4 *>(a.tiles + 4 + 4 * i);
        t->slot = w.x;
        t->first = w.y;
        t->count = w.z;
        return true;
    }
    t->first = i * QM_LORA_TILE;
    t->count = min(QM_LORA_TILE, a.tokens - t->first);
    t->slot = a.rank[0] > 0 ? 0 : -1;
    return t->count > 0;
}
__device__ __forceinline__ int64_t token_at(const QmLoraBatchArgs &a, int place) { return a.list ? a.list[place] : place; }

__device__ __forceinline__ float read_any(const void *p, int64_t i, int type) {
    if (type == 0) return reinterpret_cast<const float *>(p)[i];
    if (type == 1) return __half2float(reinterpret_cast<const __half *>(p)[i]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
}

}  // namespace

// A slot's matrices into their places, both rounded to bf16, the type the products take (float32 and float16 adapters lose
// bits here, bf16 ones none): rank by rank for what sums over the wide side, column by column for what sums over the ranks.
// Zeros behind the rank and the rows. A block takes 32 ranks x 64 columns of A or B through shared memory.
extern "C" __global__ void __launch_bounds__(256) qm_lora_set(const __grid_constant__ QmLoraSetArgs a) {
    wait_for_inputs();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *a.scale_out = a.scale;
        *a.rank_out = a.rank;
    }
    if (a.rank == 0) return;
    __shared__ uint16_t tile[32][66];
    const int tr = (a.rpad + 31) / 32, ta = (a.cols + 63) / 64, tb = (a.np + 63) / 64;
    for (int t = blockIdx.x; t < tr * (ta + tb); t += gridDim.x) {
        const int r0 = (t % tr) * 32, w = t / tr;
        const bool is_a = w < ta;
        const int c0 = (is_a ? w : w - ta) * 64, cols = is_a ? a.cols : a.rows, pitch = is_a ? a.cols : a.np;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // A lies rank by rank, B column by column: neighbouring threads read neighbours
            const int e = threadIdx.x + 256 * i;
            const int r = is_a ? e >> 6 : e & 31, c = is_a ? e & 63 : e >> 5;
            uint32_t v = 0;
            if (r0 + r < a.rank && c0 + c < cols)
                v = bf_bits(is_a ? read_any(a.a, (int64_t)(r0 + r) * a.cols + c0 + c, a.type) : read_any(a.b, (int64_t)(c0 + c) * a.rank + r0 + r, a.type));
            tile[r][c] = (uint16_t)v;
        }
        __syncthreads();
        uint16_t *by_rank = is_a ? a.da : a.db, *by_col = is_a ? a.dat : a.dbt;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = threadIdx.x + 256 * i;
            {
                const int r = e >> 5, c = (e & 31) * 2;
                if (r0 + r < a.rpad && c0 + c < pitch)
                    *reinterpret_cast<uint32_t *>(by_rank + (int64_t)(r0 + r) * pitch + c0 + c) = *reinterpret_cast<const uint32_t *>(&tile[r][c]);
            }
            {
                const int r = (e & 15) * 2, c = e >> 4;
                if (r0 + r < a.rpad && c0 + c < cols)
                    *reinterpret_cast<uint32_t *>(by_col + (int64_t)(c0 + c) * a.rpad + r0 + r) = tile[r][c] | (uint32_t)tile[r + 1][c] << 16;
            }
        }
        __syncthreads();
    }
}

// ---- 1..8 float32 rows ---------------------------------------------------------------------------------------------------
// One launch: a cluster of eight CTAs takes the rows of one adapter (the cluster of the first such row; the others leave at
// once). Each CTA multiplies an eighth of x with its columns of A, the partial sums meet in distributed shared memory, and
// each CTA then adds its own columns of B. `nsplit` clusters share the columns and repeat the first half. The first columns
// of B are on their way to shared memory while A is read.
extern "C" __global__ void __launch_bounds__(512) qm_lora_rows(const __grid_constant__ QmLoraRowsArgs a) {
    wait_for_inputs();
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cluster = blockIdx.x / QM_LORA_CLUSTER, me = (int)cluster_rank();
    const int row = cluster / a.nsplit, part = cluster % a.nsplit;
    const int np_cta = (((a.np + a.nsplit * QM_LORA_CLUSTER - 1) / (a.nsplit * QM_LORA_CLUSTER)) + 7) & ~7;
    const int n0 = min((part * QM_LORA_CLUSTER + me) * np_cta, a.rows), nn = min(np_cta, a.rows - n0);
    int slot = a.ids ? a.ids[row] : 0;
    const int r = slot >= 0 && slot < a.slots ? a.rank[slot] : 0;
    if (r == 0) {   // no adapter
        if (a.base != a.y)
            for (int c = tid; c < nn; c += 512) a.y[row * a.ldy + n0 + c] = a.base ? a.base[row * a.ldb + n0 + c] : 0.f;
        return;
    }
    int mine[8], nr = 0;   // the rows of this adapter
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const bool same = i < a.m && (a.ids ? a.ids[i] : 0) == slot;
        if (same && i < row) return;   // an earlier row's cluster has this one
        mine[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < a.m && (a.ids ? a.ids[i] : 0) == slot) {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k == nr) mine[k] = i;
            nr++;
        }
    const int ks = ((a.cols + QM_LORA_CLUSTER - 1) / QM_LORA_CLUSTER + 7) & ~7;
    const int k0 = min(me * ks, a.cols), kn = min(ks, a.cols - k0);
    float *part_u = reinterpret_cast<float *>(smem);                 // [8][rpad]
    float *u = part_u + 8 * a.rpad;                                  // [rpad][8]
    float *ssq = u + 8 * a.rpad;                                     // [8] of this CTA, then [8][16] of the warps
    uint16_t *b0 = reinterpret_cast<uint16_t *>(ssq + 8 + 128);      // [rpad][CHUNK]
    float *xs = reinterpret_cast<float *>(b0 + a.rpad * QM_LORA_CHUNK);   // [8][ks]; later the sums, then the second chunk
    float *sums = xs;                                                // [4][8][CHUNK]
    uint16_t *b1 = reinterpret_cast<uint16_t *>(xs + 32 * QM_LORA_CHUNK);
    const uint16_t *wb = a.b + (int64_t)slot * a.rpad * a.np;
    auto fetch_b = [&](int chunk) {
        const int c0 = chunk * QM_LORA_CHUNK, units = (min(QM_LORA_CHUNK, nn - c0) + 7) / 8;
        const uint32_t dst = smem_u32(chunk & 1 ? b1 : b0);
        for (int i = tid; i < r * (QM_LORA_CHUNK / 8); i += 512) {
            const int rr = i / (QM_LORA_CHUNK / 8), q = i % (QM_LORA_CHUNK / 8);
            if (q < units) copy16(dst + (rr * QM_LORA_CHUNK + q * 8) * 2, wb + (int64_t)rr * a.np + n0 + c0 + q * 8, 16);
        }
        copy_commit();
    };
    if (nn > 0) fetch_b(0);
    // x, transformed as qm_matvec stages it; the scale of a norm is one factor per row and comes in at the end
    const bool norm = a.xop == 1 || a.xop == 2;
    for (int i = 0; i < nr; i++) {
        int xr = mine[0];
#pragma unroll
        for (int k = 1; k < 8; k++) xr = k == i ? mine[k] : xr;
        const float *x = a.x + xr * a.ldx + k0, *x2 = a.x2 ? a.x2 + xr * a.ldx + k0 : nullptr;
        float ss = 0.f;
        for (int c = 4 * tid; c < kn; c += 2048) {
            float4 v = *reinterpret_cast<const float4 *>(x + c);
            if (a.xop >= 2) {
                const float4 w = *reinterpret_cast<const float4 *>(x2 + c);
                if (a.xop == 2) {
                    v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
                } else {
                    v.x = v.x / (1.f + expf(-v.x)) * w.x;
                    v.y = v.y / (1.f + expf(-v.y)) * w.y;
                    v.z = v.z / (1.f + expf(-v.z)) * w.z;
                    v.w = v.w / (1.f + expf(-v.w)) * w.w;
                }
            }
            ss += v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w;
            *reinterpret_cast<float4 *>(xs + i * ks + c) = v;
        }
        if (norm) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (lane == 0) ssq[8 + i * 16 + warp] = ss;
        }
    }
    __syncthreads();
    if (norm && tid < nr) {
        float s = 0.f;
        for (int w = 0; w < 16; w++) s += ssq[8 + tid * 16 + w];
        ssq[tid] = s;
    }
    // a warp per rank: this CTA's columns of one row of A with every activation row
    for (int rr = warp; rr < r; rr += 16) {
        const uint16_t *w = a.a + ((int64_t)slot * a.rpad + rr) * a.cols + k0;
        float acc[8];
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] = 0.f;
#pragma unroll 2
        for (int c = 8 * lane; c < kn; c += 256) {
            const uint4 q = *reinterpret_cast<const uint4 *>(w + c);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < nr) {
                    const float4 v = *reinterpret_cast<const float4 *>(xs + i * ks + c), z = *reinterpret_cast<const float4 *>(xs + i * ks + c + 4);
                    acc[i] += bf_lo(q.x) * v.x + bf_hi(q.x) * v.y + bf_lo(q.y) * v.z + bf_hi(q.y) * v.w + bf_lo(q.z) * z.x +
                              bf_hi(q.z) * z.y + bf_lo(q.w) * z.z + bf_hi(q.w) * z.w;
                }
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < nr) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
                if (lane == 0) part_u[i * a.rpad + rr] = acc[i];
            }
    }
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    // every CTA adds the eight partial sums in the same order
    const float scale = a.scale[slot];
    for (int e = tid; e < nr * r; e += 512) {
        const int i = e / r, rr = e - i * r;
        const uint32_t at = smem_u32(part_u + i * a.rpad + rr);
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < QM_LORA_CLUSTER; k++) s += peer_f32(peer_addr(at, k));
        if (norm) {
            const uint32_t sa = smem_u32(ssq + i);
            float q = 0.f;
#pragma unroll
            for (int k = 0; k < QM_LORA_CLUSTER; k++) q += peer_f32(peer_addr(sa, k));
            s *= rsqrtf(q / (float)a.cols + a.eps);
        }
        u[rr * 8 + i] = s * scale;
    }
    cluster_arrive();   // done with the others' memory; waited for before leaving
    const int group = tid >> 7, col2 = (tid & 127) * 2;
    const int chunks = (nn + QM_LORA_CHUNK - 1) / QM_LORA_CHUNK;
    for (int k = 0; k < chunks; k++) {
        copy_wait<0>();
        __syncthreads();
        if (k + 1 < chunks) fetch_b(k + 1);
        const uint16_t *b = k & 1 ? b1 : b0;
        float acc[8][2];
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i][0] = acc[i][1] = 0.f;
        for (int rr = group; rr < r; rr += 4) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(b + rr * QM_LORA_CHUNK + col2);
            const float lo = bf_lo(w), hi = bf_hi(w);
            const float4 p = *reinterpret_cast<const float4 *>(u + rr * 8), q = *reinterpret_cast<const float4 *>(u + rr * 8 + 4);
            const float v[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < nr) {
                    acc[i][0] += v[i] * lo;
                    acc[i][1] += v[i] * hi;
                }
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < nr) *reinterpret_cast<float2 *>(sums + (group * 8 + i) * QM_LORA_CHUNK + col2) = make_float2(acc[i][0], acc[i][1]);
        __syncthreads();
        const int width = min(QM_LORA_CHUNK, nn - k * QM_LORA_CHUNK);
        for (int e = tid; e < nr * QM_LORA_CHUNK; e += 512) {
            const int i = e / QM_LORA_CHUNK, c = e % QM_LORA_CHUNK;
            if (c >= width) continue;
            int yr = mine[0];
#pragma unroll
            for (int q = 1; q < 8; q++) yr = q == i ? mine[q] : yr;
            const float *s = sums + i * QM_LORA_CHUNK + c;
            const int64_t at = n0 + k * QM_LORA_CHUNK + c;
            const float d = (s[0] + s[8 * QM_LORA_CHUNK]) + (s[16 * QM_LORA_CHUNK] + s[24 * QM_LORA_CHUNK]);
            a.y[yr * a.ldy + at] = (a.base ? a.base[yr * a.ldb + at] : 0.f) + d;
        }
    }
    cluster_wait();
}

// ---- the tokens' order by adapter ----------------------------------------------------------------------------------------
// One CTA. Every warp owns a range of tokens and counts its groups; counts of the warps before and of the groups before give
// each token its place, so tokens keep their order inside a group, in every run.
extern "C" __global__ void __launch_bounds__(1024) qm_lora_lists(const __grid_constant__ QmLoraListsArgs a) {
    wait_for_inputs();
    extern __shared__ int32_t hist[];   // [32][groups], [512] tokens before, [512] tiles before
    const int groups = a.slots + 1, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int32_t *before = hist + 32 * groups, *tiles = before + 512;
    for (int i = tid; i < 32 * groups; i += 1024) hist[i] = 0;
    __syncthreads();
    const int per = ((a.tokens + 31) / 32 + 31) & ~31;
    const int t0 = warp * per, t1 = min(t0 + per, a.tokens);
    auto group_of = [&](int t) {
        const int id = a.ids[t];
        return id >= 0 && id < a.slots && a.rank[id] > 0 ? id : a.slots;
    };
    for (int t = t0; t < t1; t += 32) {
        const int g = t + lane < t1 ? group_of(t + lane) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, g);
        if (g >= 0 && lane == __ffs(same) - 1) hist[warp * groups + g] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    int total = 0;
    if (tid < groups)
        for (int w = 0; w < 32; w++) {
            const int n = hist[w * groups + tid];
            hist[w * groups + tid] = total;
            total += n;
        }
    const int mine = (total + QM_LORA_TILE - 1) / QM_LORA_TILE;
    if (tid < 512) {
        before[tid] = total;
        tiles[tid] = mine;
    }
    __syncthreads();
    for (int o = 1; o < 512; o <<= 1) {
        int p = 0, q = 0;
        if (tid < 512 && tid >= o) {
            p = before[tid - o];
            q = tiles[tid - o];
        }
        __syncthreads();
        if (tid < 512) {
            before[tid] += p;
            tiles[tid] += q;
        }
        __syncthreads();
    }
    // both are now sums up to and with the group
    const int ntiles = tiles[groups - 1];
    if (tid <= groups) a.offsets[tid] = tid ? before[tid - 1] : 0;
    if (tid == 0) a.tiles[0] = ntiles;
    for (int i = tid; i < ntiles; i += 1024) {
        int lo = 0, hi = groups - 1;   // the first group whose sum is above i
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (tiles[mid] > i) hi = mid;
            else lo = mid + 1;
        }
        const int first = (lo ? before[lo - 1] : 0) + (i - (lo ? tiles[lo - 1] : 0)) * QM_LORA_TILE;
        *reinterpret_cast<int4 *>(a.tiles + 4 + 4 * i) = make_int4(lo < a.slots ? lo : -1, first, min(QM_LORA_TILE, before[lo] - first), 0);
    }
    for (int t = t0; t < t1; t += 32) {
        const int g = t + lane < t1 ? group_of(t + lane) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, g);
        int at = 0;
        if (g >= 0) at = hist[warp * groups + g] + (g ? before[g - 1] : 0) + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (g >= 0) {
            a.list[at] = t + lane;
            if (lane == __ffs(same) - 1) hist[warp * groups + g] += __popc(same);
        }
        __syncwarp();
    }
}

// ---- shrink --------------------------------------------------------------------------------------------------------------
// A cluster of `split` CTAs takes one tile of 64 tokens of one adapter, each CTA a range of the columns, 128 per stage by
// cp.async (16-byte pieces swizzled so that ldmatrix meets no bank twice). The eight warps share the columns of a stage, not
// the tokens: every warp multiplies all 64 tokens with its 16 columns, so the tokens and the adapter are read from shared
// memory once (from 32 ranks on the warps also share the ranks, and the tokens are read two or four times). The sums meet in
// distributed shared memory and are added in a fixed order. An accumulator takes at most four products before it is added to
// a float32 sum: tensor core accumulation truncates, and a chain over all of K would carry that.
namespace {

template <int RP>
__device__ __forceinline__ void shrink(const QmLoraBatchArgs &a) {
    wait_for_inputs();
    extern __shared__ __align__(128) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int me = a.split > 1 ? (int)cluster_rank() : 0;
    const int unit = blockIdx.x / a.split;
    const QmLoraSide &s = a.side[unit < a.tiles_max ? a.first_side : 1 - a.first_side];
    Tile t;
    if (!get_tile(a, unit < a.tiles_max ? unit : unit - a.tiles_max, &t) || t.slot < 0) return;   // the whole cluster
    constexpr int R = RP * 16, STAGE = (64 + R) * 256, STAGES = QM_LORA_SHRINK_STAGES(RP);
    constexpr int WN = QM_LORA_SHRINK_GROUPS(RP), WK = 8 / WN;   // warps by rank and by column
    constexpr int NP = RP / WN;                             // pairs of n-tiles of a warp
    constexpr int SL = 8 / WK;                              // slices of 16 columns of a warp and stage
    const int wk = warp % WK, wn = warp / WK;
    const int rank = a.rank[t.slot], r16 = (rank + 15) & ~15, mt = (t.count + 15) >> 4;
    const int chunks = (s.cols + 127) / 128, per = (chunks + a.split - 1) / a.split;
    const int c0 = min(me * per, chunks), cn = min(per, chunks - c0);
    const uint32_t base = smem_u32(smem);
    // thread: piece tid % 16 of rows tid / 16 + 16 i
    const int piece = tid & 15, sub = tid >> 4;
    const uint32_t sw = (piece ^ (sub & 7)) * 16;
    const uint16_t *xrow[4];
    bool there[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = sub + 16 * i;
        there[i] = row < t.count;
        xrow[i] = s.x + token_at(a, t.first + (there[i] ? row : 0)) * s.ldx + piece * 8;
    }
    const uint16_t *w = s.w + ((int64_t)t.slot * a.rpad + sub) * s.pitch + piece * 8;
    auto fetch = [&](int chunk) {
        if (chunk < cn) {
            const uint32_t st = base + (chunk % STAGES) * STAGE;
            const int col = (c0 + chunk) * 128;
            const int left = max(0, min(16, (s.cols - col - piece * 8) * 2));   // bytes of this piece inside the rows
            // a piece behind the rows' end reads nothing, from an address that is there
            const int at = left ? col : -piece * 8;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < mt) copy16(st + (sub + 16 * i) * 256 + sw, xrow[i] + at, there[i] ? left : 0);
#pragma unroll
            for (int i = 0; i < RP; i++)
                if (16 * i < r16) copy16(st + (64 + sub + 16 * i) * 256 + sw, w + (int64_t)16 * i * s.pitch + at, left);
        }
        copy_commit();
    };
    float sum[4][2 * NP][4], acc[4][2 * NP][4];
#pragma unroll
    for (int m = 0; m < 4; m++)
#pragma unroll
        for (int n = 0; n < 2 * NP; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) sum[m][n][k] = acc[m][n][k] = 0.f;
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(i);
    for (int c = 0; c < cn; c++) {
        copy_wait<STAGES - 2>();
        __syncthreads();
        fetch(c + STAGES - 1);
        const uint32_t st = base + (c % STAGES) * STAGE;
#pragma unroll
        for (int sl = 0; sl < SL; sl++) {
            const int k = wk * SL + sl;
            uint32_t fb[NP][4];
#pragma unroll
            for (int n = 0; n < NP; n++) {
                const int wr = 64 + (wn * NP + n) * 16 + (lane & 7) + ((lane >> 4) & 1) * 8;
                ldsm4(st + wr * 256 + (((2 * k + ((lane >> 3) & 1)) ^ (wr & 7)) * 16), fb[n]);
            }
#pragma unroll
            for (int m = 0; m < 4; m++)
                if (m < mt) {
                    uint32_t fa[4];
                    const int row = m * 16 + (lane & 15);
                    ldsm4(st + row * 256 + (((2 * k + (lane >> 4)) ^ (row & 7)) * 16), fa);
#pragma unroll
                    for (int n = 0; n < NP; n++)
                        if ((wn * NP + n) * 16 < r16) {
                            mma(acc[m][2 * n], fa, fb[n][0], fb[n][1]);
                            mma(acc[m][2 * n + 1], fa, fb[n][2], fb[n][3]);
                        }
                }
        }
        if ((c & (4 / SL - 1)) == 4 / SL - 1 || c == cn - 1)
#pragma unroll
            for (int m = 0; m < 4; m++)
#pragma unroll
                for (int n = 0; n < 2 * NP; n++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        sum[m][n][k] += acc[m][n][k];
                        acc[m][n][k] = 0.f;
                    }
    }
    copy_wait<0>();
    __syncthreads();
    // [WK][64][R + 4] sums of the warps, added into the first
    float *part = reinterpret_cast<float *>(smem);
    constexpr int LD = R + 4;
    {
        const int g = lane >> 2, q = (lane & 3) * 2;
        float *p = part + wk * 64 * LD + wn * NP * 16;
#pragma unroll
        for (int m = 0; m < 4; m++)
            if (m < mt) {
#pragma unroll
                for (int n = 0; n < 2 * NP; n++) {
                    *reinterpret_cast<float2 *>(p + (m * 16 + g) * LD + n * 8 + q) = make_float2(sum[m][n][0], sum[m][n][1]);
                    *reinterpret_cast<float2 *>(p + (m * 16 + g + 8) * LD + n * 8 + q) = make_float2(sum[m][n][2], sum[m][n][3]);
                }
            }
    }
    __syncthreads();
    for (int e = tid; e < t.count * (R / 2); e += 256) {
        float *p = part + (e / (R / 2)) * LD + (e % (R / 2)) * 2;
        float2 v = *reinterpret_cast<float2 *>(p);
#pragma unroll
        for (int k = 1; k < WK; k++) {
            const float2 o = *reinterpret_cast<const float2 *>(p + k * 64 * LD);
            v.x += o.x;
            v.y += o.y;
        }
        *reinterpret_cast<float2 *>(p) = v;
    }
    __syncthreads();
    if (a.split > 1) {
        cluster_arrive();
        cluster_wait();
    }
    const float scale = a.scale[t.slot];
    // the CTAs take turns over the rows
    for (int e = tid; e < ((t.count - me + a.split - 1) / a.split) * (R / 2); e += 256) {
        const int row = me + (e / (R / 2)) * a.split, r = (e % (R / 2)) * 2;
        const uint32_t at = smem_u32(part + row * LD + r);
        float2 v = make_float2(0.f, 0.f);
        if (a.split > 1) {
            for (int k = 0; k < a.split; k++) {
                const float2 p = peer_f32x2(peer_addr(at, k));
                v.x += p.x;
                v.y += p.y;
            }
        } else {
            v = *reinterpret_cast<const float2 *>(part + row * LD + r);
        }
        uint32_t p[3], q[3];
        split3(r < rank ? v.x * scale : 0.f, p);
        split3(r + 1 < rank ? v.y * scale : 0.f, q);
        uint16_t *out = s.low + ((int64_t)t.first + row) * a.rpad + r;
#pragma unroll
        for (int k = 0; k < 3; k++) *reinterpret_cast<uint32_t *>(out + k * a.plane) = p[k] | q[k] << 16;
    }
    if (a.split > 1) {
        cluster_arrive();
        cluster_wait();
    }
}

// ---- expand --------------------------------------------------------------------------------------------------------------
// A CTA takes a tile's tokens x 256 columns, each of its eight warps 32 columns, without a barrier. All of base is asked for
// at the start (cp.async into the warp's own shared memory, no registers held); the adapter's fragments of the columns stay
// in registers while the warp goes through the tokens, 16 at a time. Both operands' fragments come straight from memory: the
// order of the ranks inside a product is free, so a lane takes eight neighbouring ranks of its token and of its column as
// one 16-byte load each. The products are added to base in shared memory and leave in rows of 128 bytes.
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <int RP, bool VEC>
__device__ __forceinline__ void expand(const QmLoraBatchArgs &a) {
    wait_for_inputs();
    extern __shared__ __align__(128) unsigned char smem[];   // [8 warps][4][16][32] floats, 16-byte pieces swizzled by the row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Tile t;
    if (!get_tile(a, blockIdx.x, &t)) return;
    const QmLoraSide &s = a.side[a.out_side];
    const int c0 = blockIdx.y * 256 + warp * 32;
    if (c0 >= s.cols) return;
    const int rank = t.slot < 0 ? 0 : a.rank[t.slot];
    if (rank == 0 && a.base == a.y) return;
    const int mt = (t.count + 15) >> 4;
    const int g = lane >> 2, q = lane & 3;
    float *own = reinterpret_cast<float *>(smem) + warp * 4 * 512;
    // (tokens of the tile: lane holds two, row l and 32 + l)
    const int tok0 = (int)token_at(a, t.first + min(lane, t.count - 1)), tok1 = (int)token_at(a, t.first + min(lane + 32, t.count - 1));
    auto token = [&](int row) { return (int64_t)__shfl_sync(0xffffffffu, row < 32 ? tok0 : tok1, row & 31); };
#pragma unroll
    for (int m = 0; m < 4; m++) {
        if (m < mt) {
            if constexpr (VEC) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = (lane >> 3) + 4 * i, piece = lane & 7, c = c0 + 4 * piece;
                    // the four rows of this step lie in one half of the tile
                    const int64_t row = __shfl_sync(0xffffffffu, m < 2 ? tok0 : tok1, (m & 1) * 16 + r);
                    const bool in = a.base && m * 16 + r < t.count && c < s.cols;
                    copy16(smem_u32(own + m * 512 + r * 32 + ((piece ^ (r & 7)) * 4)), in ? (const void *)(a.base + row * a.ldb + c) : (const void *)s.wt, in ? 16 : 0);
                }
            } else {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int64_t row = token(m * 16 + r);
                    const bool in = a.base && m * 16 + r < t.count && c0 + lane < s.cols;
                    copy4(smem_u32(own + m * 512 + r * 32 + (((lane >> 2) ^ (r & 7)) * 4) + (lane & 3)),
                          in ? (const void *)(a.base + row * a.ldb + c0 + lane) : (const void *)s.wt, in ? 4 : 0);
                }
            }
        }
        copy_commit();
    }
    constexpr int KB = RP == 1 ? 1 : RP / 2;      // groups of 32 ranks (one of 16)
    constexpr int W = RP == 1 ? 4 : 8;            // ranks of a lane
    const int kb = RP == 1 ? (rank > 0) : (rank + 31) / 32;
    auto load = [](const uint16_t *p, uint32_t (&f)[W / 2]) {
        if constexpr (W == 8) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p);
            f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            f[0] = v.x; f[1] = v.y;
        }
    };
    uint32_t fb[KB][4][W / 2];
#pragma unroll
    for (int k = 0; k < KB; k++)
#pragma unroll
        for (int n = 0; n < 4; n++)   // (a column behind the last one: any other, the result is not stored)
            if (k < kb) load(s.wt + ((int64_t)t.slot * s.cols + min(c0 + n * 8 + g, s.cols - 1)) * a.rpad + k * 32 + W * q, fb[k][n]);
    const uint16_t *low = a.side[1 - a.out_side].low + ((int64_t)t.first + g) * a.rpad + W * q;
#pragma unroll
    for (int m = 0; m < 4; m++) {
        if (m >= mt) break;
        float d[4][4];
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) d[n][k] = 0.f;
        const uint16_t *lm = low + (int64_t)m * 16 * a.rpad;
#pragma unroll
        for (int k = 0; k < KB; k++)
            if (k < kb) {
#pragma unroll
                for (int p = 2; p >= 0; p--) {   // the small parts first
                    uint32_t u0[W / 2], u1[W / 2];
                    load(lm + p * a.plane + k * 32, u0);
                    load(lm + p * a.plane + 8 * a.rpad + k * 32, u1);
#pragma unroll
                    for (int j = 0; j < W / 4; j++) {
                        const uint32_t fa[4] = {u0[2 * j], u1[2 * j], u0[2 * j + 1], u1[2 * j + 1]};
#pragma unroll
                        for (int n = 0; n < 4; n++) mma(d[n], fa, fb[k][n][2 * j], fb[k][n][2 * j + 1]);
                    }
                }
            }
        if (m == 0) copy_wait<3>();
        else if (m == 1) copy_wait<2>();
        else if (m == 2) copy_wait<1>();
        else copy_wait<0>();
        __syncwarp();
        float *st = own + m * 512;
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) {   // rows g and g + 8 share their swizzle
                float2 *p = reinterpret_cast<float2 *>(st + (g + 8 * h) * 32 + (((2 * n + (q >> 1)) ^ g) * 4) + (q & 1) * 2);
                float2 v = *p;
                v.x += d[n][2 * h];
                v.y += d[n][2 * h + 1];
                *p = v;
            }
        __syncwarp();
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = (lane >> 3) + 4 * i, piece = lane & 7, c = c0 + 4 * piece;
                const int64_t row = __shfl_sync(0xffffffffu, m < 2 ? tok0 : tok1, (m & 1) * 16 + r);
                const float4 v = *reinterpret_cast<const float4 *>(st + r * 32 + ((piece ^ (r & 7)) * 4));
                if (m * 16 + r < t.count && c < s.cols) *reinterpret_cast<float4 *>(a.y + row * a.ldy + c) = v;
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int64_t row = token(m * 16 + r);
                const float v = st[r * 32 + (((lane >> 2) ^ (r & 7)) * 4) + (lane & 3)];
                if (m * 16 + r < t.count && c0 + lane < s.cols) a.y[row * a.ldy + c0 + lane] = v;
            }
        }
    }
}

// ---- outer ---------------------------------------------------------------------------------------------------------------
// Gradient of one slot's A (or B): a cluster of `split` CTAs takes 128 columns, each CTA a range of the slot's tokens in
// stages; both operands lie token by token and enter through transposing ldmatrix. Up to 32 ranks four groups of warps share
// a stage's tokens, each with all ranks and half of the columns, so that little is read from shared memory twice; more ranks
// share the groups. The sums of the groups and of the CTAs are added in a fixed order.
template <int RP>
__device__ __forceinline__ void outer(const QmLoraBatchArgs &a) {
    wait_for_inputs();
    extern __shared__ __align__(128) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int me = a.split > 1 ? (int)cluster_rank() : 0;
    const int which = blockIdx.x / (a.outer_units * a.split), unit = blockIdx.x / a.split - which * a.outer_units;
    const QmLoraSide &s = a.side[which];
    const int blocks = (s.cols + 127) / 128;
    if (!s.grad || unit >= blocks * a.slots) return;   // the whole cluster
    const int slot = unit / blocks, n0 = (unit % blocks) * 128;
    const uint16_t *low = a.side[1 - which].low;
    const int rank = a.rank[slot], r16 = (rank + 15) & ~15;
    int first = 0, count = 0;
    if (rank > 0) {
        if (a.list) {
            first = a.offsets[slot];
            count = a.offsets[slot + 1] - first;
        } else if (slot == 0) {
            count = a.tokens;
        }
    }
    constexpr int R = RP * 16, TB = QM_LORA_OUTER_TOKENS(RP), STAGES = QM_LORA_OUTER_STAGES(RP);
    constexpr int XB = TB * 256, STAGE = XB + 3 * TB * R * 2;
    constexpr int WM = RP <= 2 ? 1 : RP / 2, WN = 2, WK = 4 / WM;   // warps by rank, by column and by token
    constexpr int MT = RP / WM, NT = 8, SL = TB / 16 / WK;
    const int chunks = (count + TB - 1) / TB, per = (chunks + a.split - 1) / a.split;
    const int c0 = min(me * per, chunks), cn = min(per, chunks - c0);
    const int wm = warp % WM, wn = warp / WM % WN, wk = warp / (WM * WN);
    const uint32_t base = smem_u32(smem);
    // tokens of the stage that is fetched next: thread's rows tid / 16 + 16 i
    int64_t tok[TB / 16];
    auto tokens_of = [&](int chunk) {
#pragma unroll
        for (int i = 0; i < TB / 16; i++) {
            const int p = (c0 + chunk) * TB + (tid >> 4) + 16 * i;
            tok[i] = chunk < cn && p < count ? token_at(a, first + p) : -1;
        }
    };
    auto fetch = [&](int chunk) {
        if (chunk < cn) {
            const uint32_t st = base + (chunk % STAGES) * STAGE;
            const int p0 = (c0 + chunk) * TB;
            const int piece = tid & 15;
#pragma unroll
            for (int i = 0; i < TB / 16; i++) {
                const int row = (tid >> 4) + 16 * i;
                const int left = tok[i] >= 0 ? max(0, min(16, (s.cols - n0 - piece * 8) * 2)) : 0;
                copy16(st + row * 256 + ((piece ^ (row & 7)) * 16), s.x + (left ? tok[i] * s.ldx + n0 + piece * 8 : 0), left);
            }
            constexpr int PIECES = R / 8;   // of a row of one plane
#pragma unroll
            for (int i = 0; i < (3 * TB * PIECES + 255) / 256; i++) {
                const int e = tid + 256 * i;
                if (3 * TB * PIECES % 256 && e >= 3 * TB * PIECES) break;
                const int plane = e / (TB * PIECES), row = (e / PIECES) % TB, piece2 = e % PIECES;
                const bool in = p0 + row < count && piece2 * 8 < r16;
                // rows of 32, 64, 128 or 256 bytes: eight rows on eight bank groups
                const int sw = PIECES >= 8 ? piece2 ^ (row & 7) : PIECES == 4 ? piece2 ^ ((row >> 1) & 3) : piece2 ^ ((row >> 2) & 1);
                copy16(st + XB + (plane * TB + row) * (R * 2) + sw * 16,
                       low + plane * a.plane + ((int64_t)first + (in ? p0 + row : 0)) * a.rpad + (in ? piece2 * 8 : 0), in ? 16 : 0);
            }
        }
        copy_commit();
    };
    float acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) acc[m][n][k] = 0.f;
    tokens_of(0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) {
        fetch(i);
        tokens_of(i + 1);
    }
    for (int c = 0; c < cn; c++) {
        copy_wait<STAGES - 2>();
        __syncthreads();
        fetch(c + STAGES - 1);
        tokens_of(c + STAGES);
        const uint32_t st = base + (c % STAGES) * STAGE;
        if (wm * MT * 16 < r16) {
#pragma unroll
            for (int sl = 0; sl < SL; sl++) {
                const int t0 = (wk * SL + sl) * 16;
                uint32_t fb[NT / 2][4];
#pragma unroll
                for (int n = 0; n < NT / 2; n++) {
                    const int row = t0 + (lane & 15);
                    ldsm4_t(st + row * 256 + ((wn * NT + 2 * n + (lane >> 4)) ^ (row & 7)) * 16, fb[n]);
                }
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int p = 2; p >= 0; p--) {   // the small parts first
                        constexpr int PIECES = R / 8;
                        uint32_t fa[4];
                        const int row = t0 + (lane >> 4) * 8 + (lane & 7), piece = (wm * MT + m) * 2 + ((lane >> 3) & 1);
                        const int sw = PIECES >= 8 ? piece ^ (row & 7) : PIECES == 4 ? piece ^ ((row >> 1) & 3) : piece ^ ((row >> 2) & 1);
                        ldsm4_t(st + XB + (p * TB + row) * (R * 2) + sw * 16, fa);
#pragma unroll
                        for (int n = 0; n < NT / 2; n++) {
                            mma(acc[m][2 * n], fa, fb[n][0], fb[n][1]);
                            mma(acc[m][2 * n + 1], fa, fb[n][2], fb[n][3]);
                        }
                    }
            }
        }
    }
    copy_wait<0>();
    __syncthreads();
    float *part = reinterpret_cast<float *>(smem);   // [WK][R][132]
    constexpr int LD = 132;
    {
        const int g = lane >> 2, q = (lane & 3) * 2;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float *p = part + (wk * R + (wm * MT + m) * 16 + g) * LD + (wn * NT + n) * 8 + q;
                *reinterpret_cast<float2 *>(p) = make_float2(acc[m][n][0], acc[m][n][1]);
                *reinterpret_cast<float2 *>(p + 8 * LD) = make_float2(acc[m][n][2], acc[m][n][3]);
            }
    }
    __syncthreads();
    if (WK > 1) {
        for (int e = tid; e < R * 64; e += 256) {
            float *p = part + (e >> 6) * LD + (e & 63) * 2;
            float2 v = *reinterpret_cast<float2 *>(p);
#pragma unroll
            for (int k = 1; k < WK; k++) {
                const float2 o = *reinterpret_cast<const float2 *>(p + k * R * LD);
                v.x += o.x;
                v.y += o.y;
            }
            *reinterpret_cast<float2 *>(p) = v;
        }
        __syncthreads();
    }
    if (a.split > 1) {
        cluster_arrive();
        cluster_wait();
    }
    // neighbouring threads take neighbours of the gradient's inner axis: columns of A, ranks of B
    float *grad = s.grad + slot * s.grad_slot;
    const int total = a.max_rank * 128, share = (total + a.split - 1) / a.split;
    for (int e = me * share + tid; e < min(total, (me + 1) * share); e += 256) {
        const int r = s.grad_col == 1 ? e >> 7 : e % a.max_rank, col = s.grad_col == 1 ? e & 127 : e / a.max_rank;
        if (n0 + col >= s.cols) continue;
        float v = 0.f;
        if (r < rank && count > 0) {
            const uint32_t at = smem_u32(part + r * LD + col);
            if (a.split > 1) {
                for (int k = 0; k < a.split; k++) v += peer_f32(peer_addr(at, k));
            } else {
                v = part[r * LD + col];
            }
        }
        grad[r * s.grad_rank + (n0 + col) * s.grad_col] = v;
    }
    if (a.split > 1) {
        cluster_arrive();
        cluster_wait();
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_shrink_r16(const __grid_constant__ QmLoraBatchArgs a) { shrink<1>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_shrink_r32(const __grid_constant__ QmLoraBatchArgs a) { shrink<2>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_shrink_r64(const __grid_constant__ QmLoraBatchArgs a) { shrink<4>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_shrink_r128(const __grid_constant__ QmLoraBatchArgs a) { shrink<8>(a); }
extern "C" __global__ void __launch_bounds__(256, 3) qm_lora_expand_r16(const __grid_constant__ QmLoraBatchArgs a) { expand<1, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 3) qm_lora_expand_r16_s(const __grid_constant__ QmLoraBatchArgs a) { expand<1, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 3) qm_lora_expand_r32(const __grid_constant__ QmLoraBatchArgs a) { expand<2, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 3) qm_lora_expand_r32_s(const __grid_constant__ QmLoraBatchArgs a) { expand<2, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 3) qm_lora_expand_r64(const __grid_constant__ QmLoraBatchArgs a) { expand<4, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 3) qm_lora_expand_r64_s(const __grid_constant__ QmLoraBatchArgs a) { expand<4, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_expand_r128(const __grid_constant__ QmLoraBatchArgs a) { expand<8, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_expand_r128_s(const __grid_constant__ QmLoraBatchArgs a) { expand<8, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_outer_r16(const __grid_constant__ QmLoraBatchArgs a) { outer<1>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_outer_r32(const __grid_constant__ QmLoraBatchArgs a) { outer<2>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_outer_r64(const __grid_constant__ QmLoraBatchArgs a) { outer<4>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_outer_r128(const __grid_constant__ QmLoraBatchArgs a) { outer<8>(a); }
