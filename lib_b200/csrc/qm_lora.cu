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

// A slot's matrices into their place: A row by row, B transposed through 32 x 32 tiles; both rounded to bf16, the type the
// products take (float32 and float16 adapters lose bits here, bf16 ones none). Zeros behind the rank and the rows.
extern "C" __global__ void __launch_bounds__(256) qm_lora_set(const __grid_constant__ QmLoraSetArgs a) {
    wait_for_inputs();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *a.scale_out = a.scale;
        *a.rank_out = a.rank;
    }
    if (a.rank == 0) return;
    const int64_t na = (int64_t)a.rpad * a.cols / 2;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < na; i += (int64_t)gridDim.x * 256) {
        const int r = (int)(2 * i / a.cols);
        uint32_t w = 0;
        if (r < a.rank) w = bf_bits(read_any(a.a, 2 * i, a.type)) | bf_bits(read_any(a.a, 2 * i + 1, a.type)) << 16;
        reinterpret_cast<uint32_t *>(a.da)[i] = w;
    }
    __shared__ uint16_t tile[32][33];
    const int tr = (a.rpad + 31) / 32, tc = (a.np + 31) / 32;
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    for (int t = blockIdx.x; t < tr * tc; t += gridDim.x) {
        const int r0 = (t % tr) * 32, n0 = (t / tr) * 32;
        for (int i = y; i < 32; i += 8)
            tile[i][x] = n0 + i < a.rows && r0 + x < a.rank ? (uint16_t)bf_bits(read_any(a.b, (int64_t)(n0 + i) * a.rank + r0 + x, a.type)) : 0;
        __syncthreads();
        for (int i = y; i < 32; i += 8)
            if (r0 + i < a.rpad && n0 + x < a.np) a.db[(int64_t)(r0 + i) * a.np + n0 + x] = tile[x][i];
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
// A cluster of `split` CTAs takes one tile of 64 tokens of one adapter, each CTA a range of the columns: four warps of 16
// tokens each, 64 columns per stage by cp.async, 16-byte pieces swizzled so that ldmatrix meets no bank twice. The sums meet
// in distributed shared memory and are added in CTA order. An accumulator takes the 64 columns of a stage and is then added
// to a float32 sum: tensor core accumulation truncates, and a chain over all of K would carry that.
namespace {
constexpr int SHRINK_STAGES = QM_LORA_SHRINK_STAGES;

template <int RP>
__device__ __forceinline__ void shrink(const QmLoraBatchArgs &a) {
    wait_for_inputs();
    extern __shared__ __align__(128) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int me = a.split > 1 ? (int)cluster_rank() : 0;
    const int unit = blockIdx.x / a.split;
    const QmLoraSide &s = a.side[unit / a.tiles_max];
    Tile t;
    if (!get_tile(a, unit % a.tiles_max, &t) || t.slot < 0) return;   // the whole cluster
    constexpr int R = RP * 16, STAGE = (64 + R) * 128;
    const int rank = a.rank[t.slot], r16 = (rank + 15) & ~15;
    const int chunks = (s.cols + 63) / 64, per = (chunks + a.split - 1) / a.split;
    const int c0 = min(me * per, chunks), cn = min(per, chunks - c0);
    const uint32_t base = smem_u32(smem);
    // thread: piece tid % 8 of rows tid / 8 + 16 i
    const int piece = tid & 7, sub = tid >> 3;
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
            const uint32_t st = base + (chunk % SHRINK_STAGES) * STAGE;
            const int col = (c0 + chunk) * 64;
            const int left = max(0, min(16, (s.cols - col - piece * 8) * 2));   // bytes of this piece inside the rows
            const uint32_t sw = (piece ^ (sub & 7)) * 16;
            // a piece behind the rows' end reads nothing, from an address that is there
            const int at = left ? col : -piece * 8;
#pragma unroll
            for (int i = 0; i < 4; i++) copy16(st + (sub + 16 * i) * 128 + sw, xrow[i] + at, there[i] ? left : 0);
#pragma unroll
            for (int i = 0; i < RP; i++)
                if (16 * i < r16) copy16(st + (64 + sub + 16 * i) * 128 + sw, w + (int64_t)16 * i * s.pitch + at, left);
        }
        copy_commit();
    };
    float sum[2 * RP][4];
#pragma unroll
    for (int n = 0; n < 2 * RP; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) sum[n][k] = 0.f;
#pragma unroll
    for (int i = 0; i < SHRINK_STAGES - 1; i++) fetch(i);
    for (int c = 0; c < cn; c++) {
        copy_wait<SHRINK_STAGES - 2>();
        __syncthreads();
        fetch(c + SHRINK_STAGES - 1);
        const uint32_t st = base + (c % SHRINK_STAGES) * STAGE;
        float acc[2 * RP][4];
#pragma unroll
        for (int n = 0; n < 2 * RP; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) acc[n][k] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            uint32_t fa[4];
            const int row = warp * 16 + (lane & 15);
            ldsm4(st + row * 128 + (((2 * k + (lane >> 4)) ^ (row & 7)) * 16), fa);
#pragma unroll
            for (int n = 0; n < RP; n++)
                if (16 * n < r16) {
                    uint32_t fb[4];
                    const int wr = n * 16 + (lane & 7) + ((lane >> 4) & 1) * 8;
                    ldsm4(st + (64 + wr) * 128 + (((2 * k + ((lane >> 3) & 1)) ^ (wr & 7)) * 16), fb);
                    mma(acc[2 * n], fa, fb[0], fb[1]);
                    mma(acc[2 * n + 1], fa, fb[2], fb[3]);
                }
        }
#pragma unroll
        for (int n = 0; n < 2 * RP; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) sum[n][k] += acc[n][k];
    }
    copy_wait<0>();
    __syncthreads();
    float *part = reinterpret_cast<float *>(smem);   // [64][R + 4]
    constexpr int LD = R + 4;
    {
        const int g = lane >> 2, q = (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < 2 * RP; n++) {
            *reinterpret_cast<float2 *>(part + (warp * 16 + g) * LD + n * 8 + q) = make_float2(sum[n][0], sum[n][1]);
            *reinterpret_cast<float2 *>(part + (warp * 16 + g + 8) * LD + n * 8 + q) = make_float2(sum[n][2], sum[n][3]);
        }
    }
    __syncthreads();
    if (a.split > 1) {
        cluster_arrive();
        cluster_wait();
    }
    const float scale = a.scale[t.slot];
    const int rows = 64 / a.split;
    for (int e = tid; e < rows * (R / 2); e += 128) {
        const int row = me * rows + e / (R / 2), r = (e % (R / 2)) * 2;
        if (row >= t.count) continue;
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
// A CTA takes 64 tokens x 128 columns: eight warps of 16 x 64. The token side's fragments come straight from the workspace
// (each is used by one warp), w's tile through shared memory; base is on its way while both arrive.
template <int RP>
__device__ __forceinline__ void expand(const QmLoraBatchArgs &a) {
    wait_for_inputs();
    extern __shared__ __align__(128) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    Tile t;
    if (!get_tile(a, blockIdx.x, &t)) return;
    const QmLoraSide &s = a.side[a.out_side];
    const int n0 = blockIdx.y * 128;
    const int wm = (warp & 3) * 16, wn = (warp >> 2) * 64;
    const int g = lane >> 2, q = (lane & 3) * 2;
    int64_t row[2];
    bool there[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        there[h] = wm + g + 8 * h < t.count;
        row[h] = token_at(a, t.first + (there[h] ? wm + g + 8 * h : 0));
    }
    const int rank = t.slot < 0 ? 0 : a.rank[t.slot], r16 = (rank + 15) & ~15;
    if (rank == 0 && a.base == a.y) return;
    const uint32_t base = smem_u32(smem);
    for (int i = tid; i < r16 * 16; i += 256) {
        const int r = i >> 4, piece = i & 15;
        const int left = max(0, min(16, (s.cols - n0 - piece * 8) * 2));
        copy16(base + r * 256 + ((piece ^ (r & 7)) * 16), s.w + ((int64_t)t.slot * a.rpad + r) * s.pitch + (left ? n0 + piece * 8 : 0), left);
    }
    copy_commit();
    float acc[8][4];
#pragma unroll
    for (int n = 0; n < 8; n++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int c = n0 + wn + n * 8 + q;
            float2 v = make_float2(0.f, 0.f);
            if (a.base && there[h]) {
                const float *p = a.base + row[h] * a.ldb + c;
                if (a.vec && c + 1 < s.cols) v = *reinterpret_cast<const float2 *>(p);
                else {
                    if (c < s.cols) v.x = p[0];
                    if (c + 1 < s.cols) v.y = p[1];
                }
            }
            acc[n][2 * h] = v.x;
            acc[n][2 * h + 1] = v.y;
        }
    float d[8][4];
#pragma unroll
    for (int n = 0; n < 8; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) d[n][k] = 0.f;
    const uint16_t *low = a.side[1 - a.out_side].low;
    copy_wait<0>();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RP; k++) {
        if (16 * k >= r16) break;
        uint32_t fa[3][4];
#pragma unroll
        for (int p = 0; p < 3; p++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int h = j & 1, r = k * 16 + (j >> 1) * 8 + q;
                fa[p][j] = there[h] ? *reinterpret_cast<const uint32_t *>(low + p * a.plane + ((int64_t)t.first + wm + g + 8 * h) * a.rpad + r) : 0u;
            }
#pragma unroll
        for (int n = 0; n < 4; n++) {
            uint32_t fb[4];
            const int wr = k * 16 + (lane & 15);
            ldsm4_t(base + wr * 256 + ((((wn >> 3) + 2 * n + (lane >> 4)) ^ (wr & 7)) * 16), fb);
#pragma unroll
            for (int p = 2; p >= 0; p--) {   // the small parts first
                mma(d[2 * n], fa[p], fb[0], fb[1]);
                mma(d[2 * n + 1], fa[p], fb[2], fb[3]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < 8; n++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int c = n0 + wn + n * 8 + q;
            if (!there[h]) continue;
            float *p = a.y + row[h] * a.ldy + c;
            const float2 v = make_float2(acc[n][2 * h] + d[n][2 * h], acc[n][2 * h + 1] + d[n][2 * h + 1]);
            if (a.vec && c + 1 < s.cols) *reinterpret_cast<float2 *>(p) = v;
            else {
                if (c < s.cols) p[0] = v.x;
                if (c + 1 < s.cols) p[1] = v.y;
            }
        }
}

// ---- outer ---------------------------------------------------------------------------------------------------------------
// Gradient of one slot's A (or B): a cluster of `split` CTAs takes 128 columns, each CTA a range of the slot's tokens in
// stages of 32; both operands lie token by token and enter through transposing ldmatrix. The CTAs' sums are added in order.
constexpr int OUTER_STAGES = QM_LORA_OUTER_STAGES;

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
    constexpr int R = RP * 16, XB = 32 * 256, STAGE = XB + 3 * 32 * R * 2;
    constexpr int WM = RP, WN = 8 / RP, NT = 128 / WN / 8;   // warps by rank and by column, n-tiles of a warp
    const int chunks = (count + 31) / 32, per = (chunks + a.split - 1) / a.split;
    const int c0 = min(me * per, chunks), cn = min(per, chunks - c0);
    const int wm = warp % WM, wn = warp / WM;
    const uint32_t base = smem_u32(smem);
    auto fetch = [&](int chunk) {
        if (chunk < cn) {
            const uint32_t st = base + (chunk % OUTER_STAGES) * STAGE;
            const int p0 = (c0 + chunk) * 32;
#pragma unroll
            for (int i = 0; i < 2; i++) {   // 32 tokens x 16 pieces
                const int e = tid + 256 * i, row = e >> 4, piece = e & 15;
                const int left = p0 + row < count ? max(0, min(16, (s.cols - n0 - piece * 8) * 2)) : 0;
                const int64_t tok = token_at(a, first + (p0 + row < count ? p0 + row : 0));
                copy16(st + row * 256 + ((piece ^ (row & 7)) * 16), s.x + tok * s.ldx + (left ? n0 + piece * 8 : 0), left);
            }
            constexpr int PIECES = R / 8;   // of a row of one plane
            for (int e = tid; e < 3 * 32 * PIECES; e += 256) {
                const int plane = e / (32 * PIECES), row = (e / PIECES) % 32, piece = e % PIECES;
                const bool in = p0 + row < count && piece * 8 < r16;
                // rows of 32, 64, 128 or 256 bytes: eight rows on eight bank groups
                const int sw = PIECES >= 8 ? piece ^ (row & 7) : PIECES == 4 ? piece ^ ((row >> 1) & 3) : piece ^ ((row >> 2) & 1);
                copy16(st + XB + (plane * 32 + row) * (R * 2) + sw * 16,
                       low + plane * a.plane + ((int64_t)first + (in ? p0 + row : 0)) * a.rpad + (in ? piece * 8 : 0), in ? 16 : 0);
            }
        }
        copy_commit();
    };
    float sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) sum[n][k] = 0.f;
#pragma unroll
    for (int i = 0; i < OUTER_STAGES - 1; i++) fetch(i);
    for (int c = 0; c < cn; c++) {
        copy_wait<OUTER_STAGES - 2>();
        __syncthreads();
        fetch(c + OUTER_STAGES - 1);
        const uint32_t st = base + (c % OUTER_STAGES) * STAGE;
        if (wm * 16 < r16) {
            float acc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) acc[n][k] = 0.f;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                uint32_t fa[3][4];
#pragma unroll
                for (int p = 0; p < 3; p++) {
                    constexpr int PIECES = R / 8;
                    const int row = k * 16 + (lane >> 4) * 8 + (lane & 7), piece = wm * 2 + ((lane >> 3) & 1);
                    const int sw = PIECES >= 8 ? piece ^ (row & 7) : PIECES == 4 ? piece ^ ((row >> 1) & 3) : piece ^ ((row >> 2) & 1);
                    ldsm4_t(st + XB + (p * 32 + row) * (R * 2) + sw * 16, fa[p]);
                }
#pragma unroll
                for (int n = 0; n < NT / 2; n++) {
                    uint32_t fb[4];
                    const int row = k * 16 + (lane & 15);
                    ldsm4_t(st + row * 256 + ((wn * NT + 2 * n + (lane >> 4)) ^ (row & 7)) * 16, fb);
#pragma unroll
                    for (int p = 2; p >= 0; p--) {
                        mma(acc[2 * n], fa[p], fb[0], fb[1]);
                        mma(acc[2 * n + 1], fa[p], fb[2], fb[3]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) sum[n][k] += acc[n][k];
        }
    }
    copy_wait<0>();
    __syncthreads();
    float *part = reinterpret_cast<float *>(smem);   // [R][132]
    constexpr int LD = 132;
    {
        const int g = lane >> 2, q = (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int col = (wn * NT + n) * 8 + q;
            *reinterpret_cast<float2 *>(part + (wm * 16 + g) * LD + col) = make_float2(sum[n][0], sum[n][1]);
            *reinterpret_cast<float2 *>(part + (wm * 16 + g + 8) * LD + col) = make_float2(sum[n][2], sum[n][3]);
        }
    }
    __syncthreads();
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

extern "C" __global__ void __launch_bounds__(128) qm_lora_shrink_r16(const __grid_constant__ QmLoraBatchArgs a) { shrink<1>(a); }
extern "C" __global__ void __launch_bounds__(128) qm_lora_shrink_r32(const __grid_constant__ QmLoraBatchArgs a) { shrink<2>(a); }
extern "C" __global__ void __launch_bounds__(128) qm_lora_shrink_r64(const __grid_constant__ QmLoraBatchArgs a) { shrink<4>(a); }
extern "C" __global__ void __launch_bounds__(128) qm_lora_shrink_r128(const __grid_constant__ QmLoraBatchArgs a) { shrink<8>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_expand_r16(const __grid_constant__ QmLoraBatchArgs a) { expand<1>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_expand_r32(const __grid_constant__ QmLoraBatchArgs a) { expand<2>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_expand_r64(const __grid_constant__ QmLoraBatchArgs a) { expand<4>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_expand_r128(const __grid_constant__ QmLoraBatchArgs a) { expand<8>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_outer_r16(const __grid_constant__ QmLoraBatchArgs a) { outer<1>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_outer_r32(const __grid_constant__ QmLoraBatchArgs a) { outer<2>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_outer_r64(const __grid_constant__ QmLoraBatchArgs a) { outer<4>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_outer_r128(const __grid_constant__ QmLoraBatchArgs a) { outer<8>(a); }
