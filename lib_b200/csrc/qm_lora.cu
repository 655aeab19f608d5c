// qm_lora.cu — low-rank adapters of many requests at once beside a shared projection, for sm_100a.
//
//   y[t] = base[t] + s B (A f(x[t])) with the A, B and s of token t's adapter; tokens without one keep their base row.
//   Backward: u = s A x, v = s B^T dy, dx = base + A^T v, dA = sum_t v x^T, dB = sum_t dy u^T over an adapter's tokens.
//
// Everything is a product with a matrix of at most 128 rows, so what bounds it is the wide side: x, base and y, dy, dx. Three
// kinds of products cover both directions:
//   shrink  low[t][r]  = sum_c x[t][c] w[r][c]   (x with A; dy with the transposed B)
//   expand  y[t][c]    = base[t][c] + sum_r low[t][r] w[r][c]
//   outer   grad[r][c] = sum_t low[t][r] x[t][c]
// The 16-bit operands are multiplied as they are. low is a float32 sum; where it is an operand it is taken as the sum of
// three bf16 (8 bits each: all 24 bits of the value), one product for each, so no rounding to 16 bits enters a result.
//
// Forms: qm_lora_rows for 1..8 float32 rows and qm_lora_few_* for up to 128 bf16 tokens do shrink and expand in one launch;
// beyond, and in the backward pass, qm_lora_lists orders the tokens by adapter and shrink, expand and outer are launches of
// their own. Measured on one B200, calls back to back, floor = what has to move at the measured copy rate of 6.54 TB/s:
//   1 row, 4096 x 4096, rank 16                       5.5 us   floor 0.05 (launch, five dependent trips to memory)
//   8 rows, 8 adapters, 6144 x 4096, rank 64          9.0 us   floor 1.4  (the same, 160 KiB of A and B per CTA)
//   64 tokens, 32 adapters, 6144 x 4096, rank 16      9.3 us   floor 1.9
//   391 tokens, 28672 x 4096, rank 32                  35 us   floor 15   (expand: base in, y out)
//   2048 tokens, 4096 x 14336, rank 64                 48 us   floor 22
//   backward, 777 tokens, 6144 x 4096, rank 8          44 us   floor 6.5  (six short launches)
//   backward, 4096 tokens, 28672 x 4096, rank 32      150 us   floor 63   (dy is read twice: 235 MB more)
#include <cuda.h>
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
// Sum over the first `split` CTAs of the cluster, in their order, of the float4 at this address of each; all are asked for
// before the first is added.
__device__ __forceinline__ float4 peers_sum4(uint32_t addr, int split) {
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k < split)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v[k].x), "=f"(v[k].y), "=f"(v[k].z), "=f"(v[k].w) : "r"(peer_addr(addr, k)) : "memory");
    }
    float4 s = v[0];
#pragma unroll
    for (int k = 1; k < 8; k++) {
        s.x += v[k].x; s.y += v[k].y; s.z += v[k].z; s.w += v[k].w;
    }
    return s;
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
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t bf_bits(float v) { return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)); }

// v as a sum of three bf16: the next 8 bits of what the ones before leave, cut off and not rounded, so that all parts have v's
// sign and none is beyond its range. Beside an infinite factor each of them has to give that infinity: an infinite v is
// infinite in all parts, and a part without bits is the smallest number there is (2^-133; not beside values below 2^-80, of
// which that would be a share that counts).
__device__ __forceinline__ void split3(float v, uint32_t (&p)[3]) {
    p[0] = __float_as_uint(v) >> 16;
    float rest = v - __uint_as_float(p[0] << 16);
    p[1] = __float_as_uint(rest) >> 16;
    rest -= __uint_as_float(p[1] << 16);
    p[2] = __float_as_uint(rest) >> 16;
    const uint32_t least = fabsf(v) >= 0x1p-80f ? (p[0] & 0x8000u) | 1u : 0u;
    if (p[1] == 0) p[1] = least;
    if (p[2] == 0) p[2] = least;
    if (!isfinite(v)) p[0] = p[1] = p[2] = bf_bits(v);
}

struct Tile {
    int slot, first, count, row, rank;   // slot -1: no adapter; count 0: no tile
};

__device__ __forceinline__ Tile get_tile(const QmLoraBatchArgs &a, int i) {
    Tile t;
    if (a.list) {
        const int4 w = *reinterpret_cast<const int4 *>(a.tiles + 8 * i);
        t.slot = w.x;
        t.first = w.y;
        t.count = w.z;
        t.row = w.w;
        t.rank = a.tiles[8 * i + 4];
    } else {
        t.rank = a.rank[0];
        t.slot = t.rank > 0 ? 0 : -1;
        t.first = t.row = i * QM_LORA_TILE;
        t.count = min(QM_LORA_TILE, a.tokens - t.first);
    }
    return t;
}
__device__ __forceinline__ int token_at(const QmLoraBatchArgs &a, int place) { return a.list ? a.list[place] : place; }

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
                // pairs of ranks in the order that expand's lanes take them: of 32 ranks (of 16, where there are no more)
                // lane q reads the pairs q, q + 4, q + 8, ... as one piece
                const int i2 = e & 15, c = e >> 4, groups = min(4, a.rpad / 8), r = (i2 % groups * 4 + i2 / groups) * 2;
                if (r0 + 2 * i2 < a.rpad && c0 + c < cols)
                    *reinterpret_cast<uint32_t *>(by_col + (int64_t)(c0 + c) * a.rpad + r0 + 2 * i2) = tile[r][c] | (uint32_t)tile[r + 1][c] << 16;
            }
        }
        __syncthreads();
    }
}

// ---- 1..8 float32 rows ---------------------------------------------------------------------------------------------------
// One launch: the rows with one id are an item, and as many clusters of eight
// CTAs as run at once are dealt to the items, which every CTA finds from the ids; the clusters of an item share its columns.
// Each CTA multiplies an eighth of x with its columns of A, the partial sums meet in distributed shared memory, and each CTA
// then adds its own columns of B. At these sizes only trips to memory count: the first columns of B and of base are on their
// way before A is read, and a warp asks for up to four ranks of A at a time.
namespace {

struct RowsShared {
    float *part;     // [8][rpad] this CTA's sums
    float *u;        // [rpad][8]
    float *ssq;      // [8]
    uint16_t *b0, *b1;   // [rpad][CHUNK]
    float *xs;       // [8][ks]; later the sums, then the second chunk of B
    float *sums;     // [4][8][CHUNK]
};

// This CTA's columns of A with NR rows of x: a warp takes ranks warp, warp + 16, ..., four of them at a time.
template <int NR>
__device__ __forceinline__ void rows_narrow(const QmLoraRowsArgs &a, const RowsShared &sh, const uint16_t *w, int r, int nr, int ks, int kn) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r0 = warp; r0 < r; r0 += 64) {
        float acc[4][NR];
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < NR; i++) acc[j][i] = 0.f;
#pragma unroll 2
        for (int c = 8 * lane; c < kn; c += 256) {
            uint4 q[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (r0 + 16 * j < r) q[j] = *reinterpret_cast<const uint4 *>(w + (int64_t)(r0 + 16 * j) * a.cols + c);
#pragma unroll
            for (int i = 0; i < NR; i++)
                if (i < nr) {
                    const float4 v = *reinterpret_cast<const float4 *>(sh.xs + i * ks + c), z = *reinterpret_cast<const float4 *>(sh.xs + i * ks + c + 4);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (r0 + 16 * j < r)
                            acc[j][i] += bf_lo(q[j].x) * v.x + bf_hi(q[j].x) * v.y + bf_lo(q[j].y) * v.z + bf_hi(q[j].y) * v.w + bf_lo(q[j].z) * z.x +
                                         bf_hi(q[j].z) * z.y + bf_lo(q[j].w) * z.z + bf_hi(q[j].w) * z.w;
                }
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (r0 + 16 * j < r) {
#pragma unroll
                for (int i = 0; i < NR; i++)
                    if (i < nr) {
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) acc[j][i] += __shfl_xor_sync(0xffffffffu, acc[j][i], o);
                        if (lane == 0) sh.part[i * a.rpad + r0 + 16 * j] = acc[j][i];
                    }
            }
    }
}

// Sums over the ranks for one chunk of columns: four groups of 128 threads share the ranks, a thread has two columns.
template <int NR>
__device__ __forceinline__ void rows_wide(const RowsShared &sh, const uint16_t *b, int r, int nr) {
    const int group = threadIdx.x >> 7, col2 = (threadIdx.x & 127) * 2;
    float acc[NR][2];
#pragma unroll
    for (int i = 0; i < NR; i++) acc[i][0] = acc[i][1] = 0.f;
#pragma unroll 4
    for (int rr = group; rr < r; rr += 4) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(b + rr * QM_LORA_CHUNK + col2);
        const float lo = bf_lo(w), hi = bf_hi(w);
        float v[NR];
        if constexpr (NR == 1) {
            v[0] = sh.u[rr * 8];
        } else {
#pragma unroll
            for (int i = 0; i < NR; i += 2) {
                const float2 p = *reinterpret_cast<const float2 *>(sh.u + rr * 8 + i);
                v[i] = p.x;
                v[i + 1] = p.y;
            }
        }
#pragma unroll
        for (int i = 0; i < NR; i++)
            if (i < nr) {
                acc[i][0] += v[i] * lo;
                acc[i][1] += v[i] * hi;
            }
    }
#pragma unroll
    for (int i = 0; i < NR; i++)
        if (i < nr) *reinterpret_cast<float2 *>(sh.sums + (group * 8 + i) * QM_LORA_CHUNK + col2) = make_float2(acc[i][0], acc[i][1]);
}

}  // namespace

extern "C" __global__ void __launch_bounds__(512) qm_lora_rows(const __grid_constant__ QmLoraRowsArgs a) {
    wait_for_inputs();
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int me = (int)cluster_rank();
    // every lane of every warp: its row's adapter, the rows that share it, and whether the row is the first of them (worked
    // out while the adapter's rank is on its way)
    const int id = lane < a.m ? (a.ids ? a.ids[lane] : 0) : -1;
    const int lane_rank = id >= 0 && id < a.slots ? a.rank[id] : 0;
    uint32_t equal = 0;
    if (lane < a.m) equal = __match_any_sync((1u << a.m) - 1, id);
    const uint32_t first = __ballot_sync(0xffffffffu, lane < a.m && __ffs(equal) - 1 == lane);
    const int items = __popc(first), parts = a.parts[items - 1];
    int item = 0, part = blockIdx.x / QM_LORA_CLUSTER;
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (part >= parts) {
            part -= parts;
            item++;
        }
    if (item >= items) return;   // the whole cluster
    uint32_t behind = first;
#pragma unroll
    for (int k = 0; k < 7; k++)
        if (k < item) behind &= behind - 1;
    const int row = __ffs(behind) - 1;
    const int slot = __shfl_sync(0xffffffffu, id, row), r = __shfl_sync(0xffffffffu, lane_rank, row);
    const uint32_t same = __shfl_sync(0xffffffffu, equal, row);   // the rows of this adapter
    const int np_cta = a.width[items - 1];
    const int n0 = min((part * QM_LORA_CLUSTER + me) * np_cta, a.rows), nn = min(np_cta, a.rows - n0);
    if (r == 0) {   // no adapter
        if (a.base != a.y)
            for (int i = 0; i < a.m; i++)
                if (same >> i & 1)
                    for (int c = tid; c < nn; c += 512) a.y[i * a.ldy + n0 + c] = a.base ? a.base[i * a.ldb + n0 + c] : 0.f;
        return;
    }
    const int nr = __popc(same);
    auto row_of = [&](int i) {   // the i-th row of this adapter
        uint32_t left = same;
#pragma unroll
        for (int k = 0; k < 7; k++)
            if (k < i) left &= left - 1;
        return __ffs(left) - 1;
    };
    const float scale = a.scale[slot];
    const int ks = ((a.cols + QM_LORA_CLUSTER - 1) / QM_LORA_CLUSTER + 7) & ~7;
    const int k0 = min(me * ks, a.cols), kn = min(ks, a.cols - k0);
    RowsShared sh;
    sh.part = reinterpret_cast<float *>(smem);
    sh.u = sh.part + 8 * a.rpad;
    sh.ssq = sh.u + 8 * a.rpad;
    sh.b0 = reinterpret_cast<uint16_t *>(sh.ssq + 8);
    sh.xs = sh.sums = reinterpret_cast<float *>(sh.b0 + a.rpad * QM_LORA_CHUNK);
    sh.b1 = reinterpret_cast<uint16_t *>(sh.xs + 32 * QM_LORA_CHUNK);
    const uint16_t *wb = a.b + (int64_t)slot * a.rpad * a.np;
    auto fetch_b = [&](int chunk) {
        const int c0 = chunk * QM_LORA_CHUNK, units = (min(QM_LORA_CHUNK, nn - c0) + 7) / 8;
        const uint32_t dst = smem_u32(chunk & 1 ? sh.b1 : sh.b0);
        for (int i = tid; i < r * (QM_LORA_CHUNK / 8); i += 512) {
            const int rr = i / (QM_LORA_CHUNK / 8), q = i % (QM_LORA_CHUNK / 8);
            if (q < units) copy16(dst + (rr * QM_LORA_CHUNK + q * 8) * 2, wb + (int64_t)rr * a.np + n0 + c0 + q * 8, 16);
        }
        copy_commit();
    };
    // this thread's outputs of a chunk: rows tid / 256 + 2 i of the adapter's, column tid % 256
    float base[4];
    const int out_col = tid % QM_LORA_CHUNK, out_row = tid / QM_LORA_CHUNK;
    auto fetch_base = [&](int chunk) {
        const int c = chunk * QM_LORA_CHUNK + out_col;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            base[i] = 0.f;
            if (a.base && out_row + 2 * i < nr && c < nn) base[i] = a.base[row_of(out_row + 2 * i) * a.ldb + n0 + c];
        }
    };
    if (nn > 0) fetch_b(0);
    // x, transformed as qm_matvec stages it; the scale of a norm is one factor per row and comes in at the end
    const bool norm = a.xop == 1 || a.xop == 2;
#pragma unroll 2
    for (int e = tid; e < nr * (kn / 4); e += 512) {
        const int i = e / (kn / 4), c = (e - i * (kn / 4)) * 4;
        const int64_t at = row_of(i) * a.ldx + k0 + c;
        float4 v = *reinterpret_cast<const float4 *>(a.x + at);
        if (a.xop >= 2) {
            const float4 w = *reinterpret_cast<const float4 *>(a.x2 + at);
            if (a.xop == 2) {
                v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
            } else {
                v.x = v.x / (1.f + expf(-v.x)) * w.x;
                v.y = v.y / (1.f + expf(-v.y)) * w.y;
                v.z = v.z / (1.f + expf(-v.z)) * w.z;
                v.w = v.w / (1.f + expf(-v.w)) * w.w;
            }
        }
        *reinterpret_cast<float4 *>(sh.xs + i * ks + c) = v;
    }
    if (nn > 0) fetch_base(0);
    __syncthreads();
    const uint16_t *wa = a.a + (int64_t)slot * a.rpad * a.cols + k0;
    if (nr == 1) rows_narrow<1>(a, sh, wa, r, nr, ks, kn);
    else if (nr == 2) rows_narrow<2>(a, sh, wa, r, nr, ks, kn);
    else if (nr <= 4) rows_narrow<4>(a, sh, wa, r, nr, ks, kn);
    else rows_narrow<8>(a, sh, wa, r, nr, ks, kn);
    if (norm && 15 - warp < nr) {   // the warps with the fewest ranks add the squares
        const int i = 15 - warp;
        float ss = 0.f;
        for (int c = 4 * lane; c < kn; c += 128) {
            const float4 v = *reinterpret_cast<const float4 *>(sh.xs + i * ks + c);
            ss += v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (lane == 0) sh.ssq[i] = ss;
    }
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    // every CTA adds the eight partial sums in the same order
    for (int e = tid; e < nr * r; e += 512) {
        const int i = e / r, rr = e - i * r;
        const uint32_t at = smem_u32(sh.part + i * a.rpad + rr), sa = smem_u32(sh.ssq + i);
        float p[QM_LORA_CLUSTER], q[QM_LORA_CLUSTER];
#pragma unroll
        for (int k = 0; k < QM_LORA_CLUSTER; k++) {
            p[k] = peer_f32(peer_addr(at, k));
            q[k] = norm ? peer_f32(peer_addr(sa, k)) : 0.f;
        }
        float s = 0.f, ss = 0.f;
#pragma unroll
        for (int k = 0; k < QM_LORA_CLUSTER; k++) {
            s += p[k];
            ss += q[k];
        }
        if (norm) s *= rsqrtf(ss / (float)a.cols + a.eps);
        sh.u[rr * 8 + i] = s * scale;
    }
    cluster_arrive();   // done with the others' memory; waited for before leaving
    const int chunks = (nn + QM_LORA_CHUNK - 1) / QM_LORA_CHUNK;
    for (int k = 0; k < chunks; k++) {
        copy_wait<0>();
        __syncthreads();
        if (k + 1 < chunks) fetch_b(k + 1);
        const uint16_t *b = k & 1 ? sh.b1 : sh.b0;
        if (nr == 1) rows_wide<1>(sh, b, r, nr);
        else if (nr == 2) rows_wide<2>(sh, b, r, nr);
        else if (nr <= 4) rows_wide<4>(sh, b, r, nr);
        else rows_wide<8>(sh, b, r, nr);
        __syncthreads();
        const int c = k * QM_LORA_CHUNK + out_col;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int yr = out_row + 2 * i;
            if (yr < nr && c < nn) {
                const float *s = sh.sums + yr * QM_LORA_CHUNK + out_col;
                const float d = (s[0] + s[8 * QM_LORA_CHUNK]) + (s[16 * QM_LORA_CHUNK] + s[24 * QM_LORA_CHUNK]);
                a.y[row_of(yr) * a.ldy + n0 + c] = base[i] + d;
            }
        }
        if (k + 1 < chunks) fetch_base(k + 1);
    }
    cluster_wait();
}

// ---- few bf16 tokens -----------------------------------------------------------------------------------------------------
// Decode batches of up to QM_LORA_FEW tokens in one launch, without lists or a workspace. Up to 16 tokens of one adapter are
// an item, and so are up to 16 without an adapter where base has to be copied. So there are at most as many items as tokens,
// and without ids, when all of them are alike, a sixteenth. Every CTA finds the items from the ids; each gets a cluster of
// eight CTAs, or as many as share the ones that run at once evenly, and the clusters behind the last item leave (which is not
// free: 64 tokens on 32 adapters take 9 us with 64 clusters and 14 with 128). As in qm_lora_rows a CTA multiplies an eighth of the
// columns of x with A, the sums meet in distributed shared memory and the CTA goes on with its own columns of B; the products
// are mma with fragments straight from memory (see expand), the columns of a warp's first piece of B and of base on their way
// before the sums meet. All that counts is the number of dependent trips to memory. Against the three launches of larger
// batches: 32 tokens of one adapter of rank 16, 6144 x 4096, 6.8 us instead of 14.3; 128 on 32, 9.6 instead of 18.2; 128 on
// one, 28672 x 4096, 16.3 instead of 20.8; 128 on two of rank 128 there, the one place where the order turns, 43 instead of 35.
namespace {

template <int RP, bool VEC>
__device__ __forceinline__ void few(const QmLoraFewArgs &a) {
    wait_for_inputs();
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int R = RP * 16, LD = R + 4, UB = QM_LORA_EXPAND_ROW(RP);
    constexpr int KB = RP == 1 ? 1 : RP / 2, W = RP == 1 ? 4 : 8;   // as in expand
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    float *part = reinterpret_cast<float *>(smem);                    // [8 warps][16][LD]; the first one the CTA's sum
    const uint32_t low = smem_u32(smem) + 8 * 16 * LD * 4;            // [16] rows of three parts
    // behind them: [FEW] adapters (`slots`: none), [FEW] tokens of the same adapter before, [FEW] the items' first tokens, [16]
    // the item's tokens, [8] scratch; over the sums, which come later: [4][SLOTS] tokens of a slot in a warp, [256] which slots
    // hold an adapter
    constexpr int SLOTS = 260;   // 256, one for none, whole words
    int32_t *ids = reinterpret_cast<int32_t *>(smem + 8 * 16 * LD * 4 + 16 * UB), *earlier = ids + QM_LORA_FEW, *leaders = earlier + QM_LORA_FEW;
    int32_t *rows = leaders + QM_LORA_FEW, *found = rows + 16;
    uint8_t *count = smem, *known = smem + 4 * SLOTS;
    const int me = (int)cluster_rank();
    int mine = tid < a.tokens ? (a.ids ? a.ids[tid] : 0) : -1;
    known[tid] = tid < a.slots && a.rank[tid] > 0;
    for (int i = tid; i < SLOTS; i += 256) reinterpret_cast<uint32_t *>(count)[i] = 0;
    if (tid < 16) rows[tid] = -1;
    __syncthreads();
    if (mine < 0 || mine >= a.slots || !known[mine]) mine = a.slots;
    if (tid >= a.tokens) mine = -1;
    if (tid < QM_LORA_FEW) ids[tid] = mine;
    const uint32_t same = __match_any_sync(0xffffffffu, mine);
    if (mine >= 0 && lane == __ffs(same) - 1) count[warp * SLOTS + mine] = (uint8_t)__popc(same);
    __syncthreads();
    int before = __popc(same & ((1u << lane) - 1));   // tokens of the same adapter before this one
    if (mine >= 0)
        for (int w = 0; w < warp; w++) before += count[w * SLOTS + mine];
    const bool leads = mine >= 0 && before % 16 == 0 && (mine < a.slots || a.base != a.y);
    const uint32_t vote = __ballot_sync(0xffffffffu, leads);
    if (lane == 0 && warp < 4) found[warp] = __popc(vote);
    if (tid < QM_LORA_FEW) earlier[tid] = before;
    __syncthreads();
    if (leads) {
        int number = __popc(vote & ((1u << lane) - 1));
        for (int w = 0; w < warp; w++) number += found[w];
        leaders[number] = tid;
    }
    __syncthreads();
    const int items = found[0] + found[1] + found[2] + found[3], parts = max(1, min(a.pieces, a.at_once / max(1, items)));
    const int np_cta = (((a.np + parts * QM_LORA_CLUSTER - 1) / (parts * QM_LORA_CLUSTER)) + 7) & ~7;
    const int unit = blockIdx.x / QM_LORA_CLUSTER;
    if (unit >= items * parts) return;   // the whole cluster
    const int leader = leaders[unit / parts];
    const int slot = ids[leader];
    const int n0 = min((unit % parts * QM_LORA_CLUSTER + me) * np_cta, a.rows), nn = min(np_cta, a.rows - n0);
    if (mine == slot && before >= earlier[leader] && before < earlier[leader] + 16) rows[before - earlier[leader]] = tid;
    __syncthreads();
    if (slot == a.slots) {   // no adapter: base rows, four at a time
        for (int i = 0; i < 16 && rows[i] >= 0; i += 4) {
            const int t[4] = {rows[i], rows[i + 1], rows[i + 2], rows[i + 3]};
            for (int c = tid; c < nn; c += 256) {
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = a.base && t[k] >= 0 ? a.base[t[k] * a.ldb + n0 + c] : 0.f;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (t[k] >= 0) a.y[t[k] * a.ldy + n0 + c] = v[k];
            }
        }
        return;
    }
    const int tok[2] = {rows[g], rows[g + 8]};   // the tokens of this lane's fragment rows, -1: none
    const int rank = a.rank[slot];
    const float scale = a.scale[slot];
    // narrow products: steps of 64 columns, dealt to the cluster's warps in turn; lane q has columns 16 q .. 16 q + 15 of a step
    const int steps = (a.cols + 63) / 64;
    const int nt = (rank + 7) / 8;
    float acc[2 * RP][4];
#pragma unroll
    for (int n = 0; n < 2 * RP; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) acc[n][k] = 0.f;
    const uint16_t *wa = a.a + (int64_t)slot * R * a.cols;
    for (int st = warp * QM_LORA_CLUSTER + me; st < steps; st += 8 * QM_LORA_CLUSTER) {
        const int k0 = st * 64 + 16 * q;
        const bool in = k0 < a.cols;   // (a multiple of 32: both halves of a lane's columns exist or neither)
        uint4 x[2][2];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < 2; j++)
                x[h][j] = in && tok[h] >= 0 ? *reinterpret_cast<const uint4 *>(a.x + tok[h] * a.ldx + k0 + 8 * j) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int n0t = 0; n0t < 2 * RP; n0t += 4) {
            if (n0t >= nt) break;
            uint4 w[4][2];
#pragma unroll
            for (int n = 0; n < 4; n++)
                if (n0t + n < 2 * RP)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        w[n][j] = in ? *reinterpret_cast<const uint4 *>(wa + (int64_t)((n0t + n) * 8 + g) * a.cols + k0 + 8 * j) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int n = 0; n < 4; n++)
                if (n0t + n < 2 * RP)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint32_t fa[4] = {x[0][j].x, x[1][j].x, x[0][j].y, x[1][j].y}, fc[4] = {x[0][j].z, x[1][j].z, x[0][j].w, x[1][j].w};
                        mma(acc[n0t + n], fa, w[n][j].x, w[n][j].y);
                        mma(acc[n0t + n], fc, w[n][j].z, w[n][j].w);
                    }
        }
    }
    // the first piece of this warp's columns
    float2 base[4][2];
    uint32_t fb[KB][4][W / 2];
    const int kb = RP == 1 ? 1 : (rank + 31) / 32;
    auto fetch = [&](int c0) {
#pragma unroll
        for (int n = 0; n < 4; n++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int c = c0 + n * 8 + 2 * q;
                base[n][h] = make_float2(0.f, 0.f);
                if (a.base && tok[h] >= 0) {
                    const float *p = a.base + tok[h] * a.ldb + n0 + c;
                    if (VEC && c + 1 < nn) base[n][h] = *reinterpret_cast<const float2 *>(p);
                    else {
                        if (c < nn) base[n][h].x = p[0];
                        if (c + 1 < nn) base[n][h].y = p[1];
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < KB; k++)
                if (k < kb) {
                    const uint16_t *p = a.bt + ((int64_t)slot * a.rows + min(n0 + c0 + n * 8 + g, a.rows - 1)) * R + k * 32 + W * q;
                    if constexpr (W == 8) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(p);
                        fb[k][n][0] = v.x; fb[k][n][1] = v.y; fb[k][n][2] = v.z; fb[k][n][3] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2 *>(p);
                        fb[k][n][0] = v.x; fb[k][n][1] = v.y;
                    }
                }
        }
    };
    if (warp * 32 < nn) fetch(warp * 32);
#pragma unroll
    for (int n = 0; n < 2 * RP; n++) {
        float *p = part + (warp * 16 + g) * LD + n * 8 + 2 * q;
        *reinterpret_cast<float2 *>(p) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2 *>(p + 8 * LD) = make_float2(acc[n][2], acc[n][3]);
    }
    __syncthreads();
    for (int e = tid; e < 16 * (R / 4); e += 256) {
        float *p = part + (e / (R / 4)) * LD + (e % (R / 4)) * 4;
        float4 v = *reinterpret_cast<float4 *>(p);
#pragma unroll
        for (int w = 1; w < 8; w++) {
            const float4 o = *reinterpret_cast<const float4 *>(p + w * 16 * LD);
            v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
        }
        *reinterpret_cast<float4 *>(p) = v;
    }
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    for (int e = tid; e < 16 * (R / 4); e += 256) {
        const int row = e / (R / 4), r = (e % (R / 4)) * 4;
        const float4 v = peers_sum4(smem_u32(part + row * LD + r), QM_LORA_CLUSTER);
        uint32_t p[4][3];
        split3(r < rank ? v.x * scale : 0.f, p[0]);
        split3(r + 1 < rank ? v.y * scale : 0.f, p[1]);
        split3(r + 2 < rank ? v.z * scale : 0.f, p[2]);
        split3(r + 3 < rank ? v.w * scale : 0.f, p[3]);
        unsigned char *out = smem + 8 * 16 * LD * 4 + row * UB + r * 2;
#pragma unroll
        for (int k = 0; k < 3; k++)
            *reinterpret_cast<uint2 *>(out + k * R * 2) = make_uint2(p[0][k] | p[1][k] << 16, p[2][k] | p[3][k] << 16);
    }
    __syncthreads();
    cluster_arrive();   // done with the others' memory; waited for before leaving
    const uint32_t lm = low + (lane & 15) * UB + (lane >> 4) * 16;
    for (int c0 = warp * 32; c0 < nn; c0 += 256) {
        float d[4][4];
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) d[n][k] = 0.f;
#pragma unroll
        for (int k = 0; k < KB; k++)
            if (k < kb) {
#pragma unroll
                for (int p = 2; p >= 0; p--)   // the small parts first
#pragma unroll
                    for (int j = 0; j < W / 4; j++) {
                        uint32_t fa[4];
                        ldsm4(lm + (p * R + k * 32 + j * 16) * 2, fa);
#pragma unroll
                        for (int n = 0; n < 4; n++) mma(d[n], fa, fb[k][n][2 * j], fb[k][n][2 * j + 1]);
                    }
            }
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                d[n][2 * h] += base[n][h].x;
                d[n][2 * h + 1] += base[n][h].y;
            }
        if (c0 + 256 < nn) fetch(c0 + 256);
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int c = c0 + n * 8 + 2 * q;
                if (tok[h] < 0) continue;
                float *p = a.y + tok[h] * a.ldy + n0 + c;
                if (VEC && c + 1 < nn) *reinterpret_cast<float2 *>(p) = make_float2(d[n][2 * h], d[n][2 * h + 1]);
                else {
                    if (c < nn) p[0] = d[n][2 * h];
                    if (c + 1 < nn) p[1] = d[n][2 * h + 1];
                }
            }
    }
    cluster_wait();
}

}  // namespace

// ---- the tokens' order by adapter ----------------------------------------------------------------------------------------
// One CTA. Every warp owns a range of tokens and counts its groups; counts of the warps before and of the groups before give
// each token its place, so tokens keep their order inside a group, in every run.
extern "C" __global__ void __launch_bounds__(1024) qm_lora_lists(const __grid_constant__ QmLoraListsArgs a) {
    wait_for_inputs();
    extern __shared__ int32_t hist[];   // [32][groups], then [512] tokens, tiles and workspace blocks up to and with the group
    const int groups = a.slots + 1, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int32_t *before = hist + 32 * groups, *tiles = before + 512, *blocks = tiles + 512;
    uint8_t *known = reinterpret_cast<uint8_t *>(blocks + 512);   // [256] slots that hold an adapter
    const int per = ((a.tokens + 31) / 32 + 31) & ~31;
    const int t0 = warp * per, t1 = min(t0 + per, a.tokens);
    constexpr int AHEAD = 8;   // ids that a lane asks for at a time; the first ones stay in registers
    int ids[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) ids[i] = t0 + 32 * i + lane < t1 ? a.ids[t0 + 32 * i + lane] : -1;
    if (tid < a.slots) known[tid] = a.rank[tid] > 0;
    for (int i = tid; i < 32 * groups; i += 1024) hist[i] = 0;
    __syncthreads();
    auto group_of = [&](int id) { return id >= 0 && id < a.slots && known[id] ? id : a.slots; };
    // f(token of this lane, its group or -1, lanes of the same group), 32 tokens at a time
    auto walk = [&](auto f) {
        for (int t = t0; t < t1; t += 32 * AHEAD) {
            int more[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int u = t + 32 * i + lane;
                more[i] = t == t0 ? ids[i] : u < t1 ? a.ids[u] : -1;
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                if (t + 32 * i >= t1) break;
                const int u = t + 32 * i + lane, g = u < t1 ? group_of(more[i]) : -1;
                f(u, g, __match_any_sync(0xffffffffu, g));
            }
        }
    };
    walk([&](int, int g, uint32_t same) {
        if (g >= 0 && lane == __ffs(same) - 1) hist[warp * groups + g] += __popc(same);
        __syncwarp();
    });
    __syncthreads();
    int total = 0;
    if (tid < groups)
        for (int w = 0; w < 32; w++) {
            const int n = hist[w * groups + tid];
            hist[w * groups + tid] = total;
            total += n;
        }
    if (tid < 512) {
        before[tid] = total;
        tiles[tid] = (total + QM_LORA_TILE - 1) / QM_LORA_TILE;
        blocks[tid] = (total + QM_LORA_BLOCK - 1) / QM_LORA_BLOCK;
    }
    __syncthreads();
    for (int o = 1; o < groups; o <<= 1) {
        int p = 0, q = 0, r = 0;
        if (tid < groups && tid >= o) {
            p = before[tid - o];
            q = tiles[tid - o];
            r = blocks[tid - o];
        }
        __syncthreads();
        if (tid < groups) {
            before[tid] += p;
            tiles[tid] += q;
            blocks[tid] += r;
        }
        __syncthreads();
    }
    if (tid <= groups) {
        a.offsets[tid] = tid ? before[tid - 1] : 0;
        a.offsets[a.slots + 2 + tid] = tid ? blocks[tid - 1] * QM_LORA_BLOCK : 0;
    }
    walk([&](int u, int g, uint32_t same) {
        int at = 0;
        if (g >= 0) at = hist[warp * groups + g] + (g ? before[g - 1] : 0) + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (g >= 0) {
            a.list[at] = u;
            if (lane == __ffs(same) - 1) hist[warp * groups + g] += __popc(same);
        }
        __syncwarp();
    });
    const int ntiles = tiles[groups - 1];
    for (int i = tid; i < a.tiles_max; i += 1024) {
        int4 w = make_int4(-1, 0, 0, 0);
        int rank = 0;
        if (i < ntiles) {
            int lo = 0, hi = groups - 1;   // the first group whose sum is above i
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (tiles[mid] > i) hi = mid;
                else lo = mid + 1;
            }
            const int in = (i - (lo ? tiles[lo - 1] : 0)) * QM_LORA_TILE;
            w.y = (lo ? before[lo - 1] : 0) + in;
            w.z = min(QM_LORA_TILE, before[lo] - w.y);
            w.w = (lo ? blocks[lo - 1] * QM_LORA_BLOCK : 0) + in;
            if (lo < a.slots) {
                w.x = lo;
                rank = a.rank[lo];
            }
        }
        reinterpret_cast<int4 *>(a.tiles)[2 * i] = w;
        a.tiles[8 * i + 4] = rank;
    }
}

// A copy of bf16 rows whose addresses or pitch no tensor map takes, 16-byte aligned: a thread writes eight columns at a time.
extern "C" __global__ void __launch_bounds__(256) qm_lora_align(const __grid_constant__ QmLoraAlignArgs a) {
    wait_for_inputs();
    const int64_t pieces = a.pitch / 8, total = pieces * a.rows;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        const int64_t row = e / pieces;
        const int c = (int)(e - row * pieces) * 8;
        const uint16_t *p = a.src + row * a.ld + c;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = c + 2 * i < a.cols ? p[2 * i] : 0u, hi = c + 2 * i + 1 < a.cols ? p[2 * i + 1] : 0u;
            w[i] = lo | hi << 16;
        }
        *reinterpret_cast<uint4 *>(a.dst + row * a.pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ---- tcgen05 plumbing ----------------------------------------------------------------------------------------------------
namespace {


// Operand tiles as 128-byte rows, 16-byte pieces swizzled by the row (the 128-byte swizzle of the tensor maps). Rows along K
// (`group` is not used: the row groups lie 1024 bytes apart), or rows along M or N with 64 elements of it each, the next 64
// `group` bytes further.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t group) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(group >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// bf16 operands, float32 accumulators, M = 128.
__device__ constexpr uint32_t tc_idesc(int n, bool along_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (along_mn ? 3u << 15 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_load16(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map),
                 "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
// Four rows by their numbers into four consecutive rows; a number behind the last row brings zeros.
__device__ __forceinline__ void tma_rows4(uint32_t dst, const CUtensorMap *map, int x, const int (&y)[4], uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3])
        : "memory");
}

// Tensor core accumulation truncates: a chain of n additions was seen 3e-8 n off. So an accumulator takes PERIOD stages (16
// additions) and is then added to float32 registers while the next stages go into a second one (where tensor memory holds
// two).
constexpr int PERIOD = 4;

// A CTA's barriers, behind its stages: full and empty per stage and per accumulator; the accumulators' address; whether a wait
// was given up.
struct Pipe {
    uint32_t full, empty, acc_full, acc_empty, tmem;
    volatile uint32_t *failed;
};
// Everything that needs no input: barriers, and tensor memory. The next kernel may start only after the tensor memory of all
// CTAs is in their hands, so that none of its CTAs can hold what one of these still asks for.
template <int STAGES>
__device__ __forceinline__ Pipe pipe_open(unsigned char *bars, uint32_t cols, int readers) {
    Pipe p;
    p.full = smem_u32(bars);
    p.empty = p.full + 8 * STAGES;
    p.acc_full = p.empty + 8 * STAGES;
    p.acc_empty = p.acc_full + 16;
    p.failed = reinterpret_cast<volatile uint32_t *>(bars + 8 * (2 * STAGES + 4) + 4);
    if (threadIdx.x == 0) {
        *p.failed = 0;
        for (int s = 0; s < 2 * STAGES + 2; s++) qm::mbar_init(p.full + 8 * s, 1);
        for (int s = 0; s < 2; s++) qm::mbar_init(p.acc_empty + 8 * s, readers);
        qm::fence_barrier_init();
    }
    __syncwarp();   // the lanes of a warp are together for what is .sync.aligned
    if (threadIdx.x < 32) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(p.acc_empty + 16), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    p.tmem = *reinterpret_cast<volatile uint32_t *>(bars + 8 * (2 * STAGES + 4));
    wait_for_inputs();
    return p;
}
__device__ __forceinline__ void pipe_close(const Pipe &p, uint32_t cols) {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    __syncwarp();
    if (threadIdx.x < 32) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(p.tmem), "r"(cols) : "memory");
    }
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A wait of a whole warp. Lanes leave a bounded wait at different polls, and at its end may even get different answers: they
// take one together, so that none waits at a barrier of the warp for lanes that have given up, and are together for the
// .sync.aligned instructions that follow.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, qm::mbar_wait_bounded(bar, parity)); }
// A wait that has run out.
__device__ __forceinline__ void give_up(const Pipe &p, unsigned int *status) {
    atomicOr(status, QM_STATUS_TIMEOUT);
    *p.failed = 1;
}
// All warps are through with the stages; where a wait was given up, copies and products that are still in flight get two
// milliseconds to land before the memory they write is used for something else and given back.
__device__ __forceinline__ void pipe_done(const Pipe &p) {
    __syncthreads();
    if (*p.failed) {
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000ll) {}
    }
}
// Where a CTA that takes one piece of work after another is: stages and periods before this piece, and whether every wait has
// ended so far (after one that has not, its warp does no more).
struct Progress {
    int stages, periods;
    bool ok;
};
__device__ __forceinline__ void advance(Progress &g, int cn) {
    g.stages += cn;
    g.periods += (cn + PERIOD - 1) / PERIOD;
}
// Before the stages that ordinary loads and stores have used are filled by TMA again.
__device__ __forceinline__ void stages_used() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// The multiplying thread: stage by stage, `issue(stage address, accumulator, first of a period)`.
template <int STAGES, int NACC, class F>
__device__ __forceinline__ void pipe_multiply(const Pipe &p, Progress &g, uint32_t base, uint32_t stage_bytes, int cn, unsigned int *status, F issue) {
    for (int c = 0; c < cn && g.ok; c++) {
        const int n = g.stages + c, st = n % STAGES, period = g.periods + c / PERIOD, acc = period % NACC;
        if (c % PERIOD == 0 && period >= NACC) g.ok = qm::mbar_wait_bounded(p.acc_empty + 8 * acc, (uint32_t)(period / NACC - 1) & 1u);
        g.ok = g.ok && qm::mbar_wait_bounded(p.full + 8 * st, (uint32_t)(n / STAGES) & 1u);
        if (!g.ok) {
            give_up(p, status);
            return;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        issue(base + st * stage_bytes, acc, c % PERIOD == 0);
        tc_commit(p.empty + 8 * st);
        if (c % PERIOD == PERIOD - 1 || c == cn - 1) tc_commit(p.acc_full + 8 * acc);
    }
}
// A reading warp: adds each period's accumulator columns `first`.. to v.
template <int N, int NACC>
__device__ __forceinline__ void pipe_read(const Pipe &p, Progress &g, uint32_t acc_cols, uint32_t first, int cn, unsigned int *status, float (&v)[N]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = 0.f;
    for (int i = 0; i * PERIOD < cn && g.ok; i++) {
        const int period = g.periods + i, acc = period % NACC;
        g.ok = warp_wait(p.acc_full + 8 * acc, (uint32_t)(period / NACC) & 1u);
        if (!g.ok) {
            if (lane == 0) give_up(p, status);
            return;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int j = 0; j < N; j += 16) {
            float o[16];
            tc_load16(p.tmem + ((uint32_t)((warp & 3) * 32) << 16) + acc * acc_cols + first + j, o);
#pragma unroll
            for (int i = 0; i < 16; i++) v[j + i] += o[i];
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(p.acc_empty + 8 * acc);
    }
}
// The loading warp's view of 32 rows: lane l holds the numbers of rows 4 l .. 4 l + 3 of the tile, `there` of them exist. Its
// group of eight lanes holds 32 rows; are those that exist neighbours?
__device__ __forceinline__ bool neighbours(const int (&rows)[4], int there) {
    const int lane = threadIdx.x & 31;
    const int first = __shfl_sync(0xffffffffu, rows[0], lane & 24);
    bool ok = true;
#pragma unroll
    for (int i = 0; i < 4; i++) ok = ok && (i >= there || rows[i] == first + 4 * (lane & 7) + i);
    const uint32_t all = __ballot_sync(0xffffffffu, ok);
    return ((all >> (lane & 24)) & 0xFFu) == 0xFFu;
}

// ---- shrink --------------------------------------------------------------------------------------------------------------
// A cluster of `split` CTAs takes one tile of 128 tokens of one adapter, the CTAs taking turns over its columns, 64 per
// stage: the adapter's ranks and the tokens by TMA, 32 tokens that are neighbours as one box, others by their numbers. One
// thread issues the products (M = the tokens, N = the ranks) into tensor memory. What a CTA reads from memory is all that
// bounds it. The CTAs' sums meet in distributed shared memory and are added in a fixed order. 4096 tokens, x of 4096 and dy of
// 28672 columns, rank 32: 52 us, 5.2 TB/s (legacy mma with cp.async: 67 us, and 71 instead of 22 at 2048 tokens x 14336, rank
// 64, where its fragments kept the issue slots and the shared memory busy).
// MANY: one side, fewer clusters than there may be tiles, each takes one after another.
constexpr int SHRINK_THREADS = 192;   // four warps that read the accumulators, one that loads, one that multiplies

template <int RP, bool MANY>
__device__ __forceinline__ void shrink(const QmLoraTcArgs &ta) {
    const QmLoraBatchArgs &a = ta.b;
    extern __shared__ unsigned char smem_raw[];
    constexpr int R = RP * 16, XB = 128 * 128, STAGE = XB + R * 128, STAGES = QM_LORA_SHRINK_STAGES(RP);
    constexpr int TCOLS = 2 * R;
    unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Pipe pipe = pipe_open<STAGES>(smem + STAGES * STAGE, TCOLS, 4);
    const int me = a.split > 1 ? (int)cluster_rank() : 0;
    Progress at_now = {0, 0, true};
    int unit = blockIdx.x / a.split;
    do {
        const int side = unit < a.tiles_max ? a.first_side : 1 - a.first_side;
        const QmLoraSide &s = a.side[side];
        const Tile t = get_tile(a, unit < a.tiles_max ? unit : unit - a.tiles_max);
        if (t.count <= 0 || t.slot < 0) continue;   // the same for the whole cluster
        const int chunks = (s.cols + 63) / 64, cn = max(0, (chunks - me + a.split - 1) / a.split);
        const uint32_t base = smem_u32(smem);
        float *part = reinterpret_cast<float *>(smem);   // [128][R + 4], over the stages once they are done
        constexpr int LD = R + 4;
        float v[R];
        if (warp == 4) {
            const int there = min(4, t.count - 4 * lane);
            int rows[4];
#pragma unroll
            for (int i = 0; i < 4; i++) rows[i] = i < there ? token_at(a, t.first + 4 * lane + i) : a.tokens;
            // (a box may bring rows behind the tile's last token: rows of the product that are not read)
            const bool box = neighbours(rows, there);
            const bool one = box ? (lane & 7) == 0 && there > 0 : there > 0;
            const uint32_t bytes = __reduce_add_sync(0xffffffffu, one ? (box ? 4096u : 512u) : 0u) + R * 128;
            for (int c = 0; c < cn && at_now.ok; c++) {
                const int n = at_now.stages + c, st = n % STAGES;
                at_now.ok = n < STAGES || warp_wait(pipe.empty + 8 * st, (uint32_t)(n / STAGES - 1) & 1u);
                if (!at_now.ok) {
                    if (lane == 0) give_up(pipe, a.status);
                    break;
                }
                const uint32_t at = base + st * STAGE, bar = pipe.full + 8 * st;
                const int x = (c * a.split + me) * 64;
                if (lane == 0) {
                    qm::mbar_expect_tx(bar, bytes);
                    tma_box(at + XB, &ta.w[side], x, t.slot * a.rpad, bar);
                }
                __syncwarp();
                if (one) {
                    if (box) tma_box(at + lane * 512, &ta.rows[side], x, rows[0], bar);
                    else tma_rows4(at + lane * 512, &ta.gather[side], x, rows, bar);
                }
            }
        } else if (warp == 5) {
            if (lane == 0)
                pipe_multiply<STAGES, 2>(pipe, at_now, base, STAGE, cn, a.status, [&](uint32_t at, int acc, bool first) {
                    const uint64_t x = tile_desc(at, 16), w = tile_desc(at + XB, 16);
#pragma unroll
                    for (int k = 0; k < 4; k++)   // 16 columns = 32 bytes = 2 descriptor units
                        tc_mma(pipe.tmem + acc * R, x + 2 * k, w + 2 * k, tc_idesc(R, false), !first || k > 0);
                });
        } else {
            pipe_read<R, 2>(pipe, at_now, R, 0, cn, a.status, v);
        }
        pipe_done(pipe);
        if (warp < 4) {
#pragma unroll
            for (int i = 0; i < R; i += 4)
                *reinterpret_cast<float4 *>(part + tid * LD + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
        __syncthreads();
        if (a.split > 1) {
            cluster_arrive();
            cluster_wait();
        }
        const float scale = a.scale[t.slot];
        const int rows = (t.count + QM_LORA_BLOCK - 1) / QM_LORA_BLOCK * QM_LORA_BLOCK;   // zeros behind the tokens
        constexpr int LP = QM_LORA_PITCH(RP);
        // the CTAs take turns over the rows, a thread takes four ranks
        for (int e = tid; e < ((rows - me + a.split - 1) / a.split) * (R / 4); e += SHRINK_THREADS) {
            const int row = me + (e / (R / 4)) * a.split, r = (e % (R / 4)) * 4;
            float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row < t.count)
                w = a.split > 1 ? peers_sum4(smem_u32(part + row * LD + r), a.split) : *reinterpret_cast<const float4 *>(part + row * LD + r);
            uint32_t p[4][3];
            split3(r < t.rank ? w.x * scale : 0.f, p[0]);
            split3(r + 1 < t.rank ? w.y * scale : 0.f, p[1]);
            split3(r + 2 < t.rank ? w.z * scale : 0.f, p[2]);
            split3(r + 3 < t.rank ? w.w * scale : 0.f, p[3]);
            uint16_t *out = s.low + ((int64_t)t.row + row) * LP + r;
#pragma unroll
            for (int k = 0; k < 3; k++)
                *reinterpret_cast<uint2 *>(out + k * R) = make_uint2(p[0][k] | p[1][k] << 16, p[2][k] | p[3][k] << 16);
        }
        if (MANY) stages_used();
        if (a.split > 1) {
            cluster_arrive();
            cluster_wait();
        } else if (MANY) {
            __syncthreads();
        }
        advance(at_now, cn);
    } while (MANY && (unit += gridDim.x / a.split) < a.tiles_max);
    pipe_close(pipe, TCOLS);
}

// ---- expand --------------------------------------------------------------------------------------------------------------
// A CTA takes half a tile's tokens x 32 columns for each of its seven or eight warps: as many as leave room for a third CTA on
// the SM, beyond 32 ranks for a second one, which has its base on its way while this one multiplies (4096 tokens x 4096, rank
// 32: three CTAs of seven warps 26.5 us, two of eight 28.6; at rank 64 three would have six, 21.8 us for 2048 tokens against
// 20.5 with two of eight). All of base is asked for at the start (cp.async into the warp's own shared memory, no registers
// held), the tokens' narrow products once for the CTA; the adapter's fragments of the columns stay in registers while the warp
// goes through the tokens, 16 at a time. The products are added to base in shared memory and leave in rows of 128 bytes.
// Legacy mma on purpose: the same step by tcgen05 (operands by TMA, results through tensor memory and shared memory, 128
// columns per CTA) took 22.5 us instead of 20.5 at 2048 tokens x 4096, rank 64, and 34 instead of 22 at 391 x 28672, rank 32,
// because every CTA then waits for tensor memory and two barriers more; leaving the products out altogether saves 1 us.
// Copying base to y by the same steps takes 13.6 and 18 us (10.3 and 13.8 at the measured copy rate).
// MANY: fewer CTAs than there may be halves of tiles, each takes one after another.
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Place of column c (0..31) of row r in a warp's [16][32] floats: 16-byte pieces moved in pairs by the row, so that neither
// the fragments' accesses (four rows x 32 bytes at a time) nor whole rows meet a bank twice.
__device__ __forceinline__ int staged(int r, int c) { return r * 32 + (((c >> 2) ^ (2 * (r & 3))) << 2) + (c & 3); }

template <int RP, bool VEC, bool MANY>
__device__ __forceinline__ void expand(const QmLoraBatchArgs &a) {
    wait_for_inputs();
    extern __shared__ __align__(128) unsigned char smem[];   // [warps][4][16][32] floats, then [64] rows of narrow products
    constexpr int THREADS = QM_LORA_EXPAND_WARPS(RP) * 32, R = RP * 16, LP = QM_LORA_PITCH(RP), UB = QM_LORA_EXPAND_ROW(RP);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const QmLoraSide &s = a.side[a.out_side];
    const int c0 = blockIdx.y * THREADS + warp * 32;   // (a column per thread)
    int half = blockIdx.x;
    bool used = false;   // shared memory
    do {
        Tile t = get_tile(a, half >> 1);
        if (MANY && t.count <= 0) return;
        if (half & 1) {
            t.first += 64;
            t.row += 64;
            t.count -= 64;
        }
        t.count = min(t.count, 64);
        if (t.count <= 0) continue;
        const int rank = t.slot < 0 ? 0 : t.rank;
        if (rank == 0 && a.base == a.y) continue;
        if (MANY && used) __syncthreads();
        used = true;
        const int mt = (t.count + 15) >> 4;
        const int g = lane >> 2, q = lane & 3;
        float *own = reinterpret_cast<float *>(smem) + warp * 4 * 512;
        const uint32_t low = smem_u32(smem) + THREADS * 256;
        // the tokens' numbers: lane holds rows l and 32 + l
        const int tok0 = token_at(a, t.first + min(lane, t.count - 1)), tok1 = token_at(a, t.first + min(lane + 32, t.count - 1));
        if (rank > 0) {
            const uint16_t *src = a.side[1 - a.out_side].low + (int64_t)t.row * LP;
            for (int e = tid; e < mt * 16 * (6 * RP); e += THREADS) {   // rows of 3 R ranks: 6 RP pieces of 16 bytes
                const int row = e / (6 * RP), piece = e % (6 * RP);
                copy16(low + row * UB + piece * 16, src + row * LP + piece * 8, 16);
            }
        }
        copy_commit();
        constexpr int KB = RP == 1 ? 1 : RP / 2;      // groups of 32 ranks (one of 16)
        constexpr int W = RP == 1 ? 4 : 8;            // ranks of a lane
        const int kb = RP == 1 ? (rank > 0) : (rank + 31) / 32;
        // (asked for before base, behind which they would come last)
        uint32_t fb[KB][4][W / 2];
#pragma unroll
        for (int k = 0; k < KB; k++)
#pragma unroll
            for (int n = 0; n < 4; n++)   // (a column behind the last one: any other, the result is not stored)
                if (k < kb) {
                    const uint16_t *p = s.wt + ((int64_t)t.slot * s.cols + min(c0 + n * 8 + g, s.cols - 1)) * R + k * 32 + W * q;
                    if constexpr (W == 8) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(p);
                        fb[k][n][0] = v.x; fb[k][n][1] = v.y; fb[k][n][2] = v.z; fb[k][n][3] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2 *>(p);
                        fb[k][n][0] = v.x; fb[k][n][1] = v.y;
                    }
                }
        const bool mine = c0 < s.cols;
#pragma unroll
        for (int m = 0; m < 4; m++) {
            if (m < mt && mine) {
                if constexpr (VEC) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = (lane >> 3) + 4 * i, c = 4 * (lane & 7);
                        const int64_t row = __shfl_sync(0xffffffffu, m < 2 ? tok0 : tok1, (m & 1) * 16 + r);
                        const bool in = a.base && m * 16 + r < t.count && c0 + c < s.cols;
                        copy16(smem_u32(own + m * 512 + staged(r, c)), in ? (const void *)(a.base + row * a.ldb + c0 + c) : (const void *)s.wt, in ? 16 : 0);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int64_t row = __shfl_sync(0xffffffffu, m < 2 ? tok0 : tok1, (m & 1) * 16 + r);
                        const bool in = a.base && m * 16 + r < t.count && c0 + lane < s.cols;
                        copy4(smem_u32(own + m * 512 + staged(r, lane)), in ? (const void *)(a.base + row * a.ldb + c0 + lane) : (const void *)s.wt, in ? 4 : 0);
                    }
                }
            }
            copy_commit();
        }
        copy_wait<4>();
        __syncthreads();
        if (!mine) continue;
#pragma unroll
        for (int m = 0; m < 4; m++) {
            if (m >= mt) break;
            float d[4][4];
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) d[n][k] = 0.f;
            const uint32_t lm = low + (m * 16 + (lane & 15)) * UB + (lane >> 4) * 16;
#pragma unroll
            for (int k = 0; k < KB; k++)
                if (k < kb) {
#pragma unroll
                    for (int p = 2; p >= 0; p--)   // the small parts first
#pragma unroll
                        for (int j = 0; j < W / 4; j++) {
                            uint32_t fa[4];
                            ldsm4(lm + (p * R + k * 32 + j * 16) * 2, fa);
#pragma unroll
                            for (int n = 0; n < 4; n++) mma(d[n], fa, fb[k][n][2 * j], fb[k][n][2 * j + 1]);
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
                for (int h = 0; h < 2; h++) {
                    float2 *p = reinterpret_cast<float2 *>(st + staged(g + 8 * h, n * 8 + 2 * q));
                    float2 v = *p;
                    v.x += d[n][2 * h];
                    v.y += d[n][2 * h + 1];
                    *p = v;
                }
            __syncwarp();
            if constexpr (VEC) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = (lane >> 3) + 4 * i, c = 4 * (lane & 7);
                    const int64_t row = __shfl_sync(0xffffffffu, m < 2 ? tok0 : tok1, (m & 1) * 16 + r);
                    const float4 v = *reinterpret_cast<const float4 *>(st + staged(r, c));
                    if (m * 16 + r < t.count && c0 + c < s.cols) *reinterpret_cast<float4 *>(a.y + row * a.ldy + c0 + c) = v;
                }
            } else {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int64_t row = __shfl_sync(0xffffffffu, m < 2 ? tok0 : tok1, (m & 1) * 16 + r);
                    const float v = st[staged(r, lane)];
                    if (m * 16 + r < t.count && c0 + lane < s.cols) a.y[row * a.ldy + c0 + lane] = v;
                }
            }
        }
    } while (MANY && (half += gridDim.x) < 2 * a.tiles_max);
}

// ---- outer ---------------------------------------------------------------------------------------------------------------
// Gradient of one slot's A (or B): a cluster of `split` CTAs takes a block of columns, the CTAs taking turns over the slot's
// tokens, 64 per stage. Both operands lie token by token, which is along M and N: M = the three parts of the ranks side by
// side, as they lie in the workspace, so one product takes all of them, N = the columns. 32 tokens that are neighbours come
// as boxes, others by their numbers; behind the slot's last token come zeros. The parts, and the CTAs' sums, are added in a
// fixed order. 4096 tokens of 4096 and 28672 columns, rank 32: 61 us (legacy mma 129), about 10 of them start and end of a CTA;
// 128 column blocks leave 20 SMs to dx, which runs beside it.
template <int RP>
__device__ __forceinline__ void outer(const QmLoraTcArgs &ta) {
    const QmLoraBatchArgs &a = ta.b;
    extern __shared__ unsigned char smem_raw[];
    constexpr int R = RP * 16, G = QM_LORA_PITCH(RP) / 64, BN = QM_LORA_OUTER_COLS(RP), NG = BN / 64;
    constexpr int AB = G * 8192, STAGE = AB + NG * 8192, STAGES = QM_LORA_OUTER_STAGES(RP);
    constexpr int MM = (G + 1) / 2;                       // products of M = 128
    constexpr int NACC = 2 * MM * BN <= 512 ? 2 : 1;
    constexpr int READERS = QM_LORA_OUTER_READERS(RP), THREADS = (READERS + 2) * 32;
    constexpr int MINE = MM * BN / (READERS / 4);         // columns of the accumulators that a reading warp adds up
    constexpr int TCOLS = 512;
    unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Pipe pipe = pipe_open<STAGES>(smem + STAGES * STAGE, TCOLS, READERS);
    const int me = a.split > 1 ? (int)cluster_rank() : 0;
    const int which = blockIdx.x / (a.outer_units * a.split), unit = blockIdx.x / a.split - which * a.outer_units;
    const QmLoraSide &s = a.side[which];
    const int blocks = (s.cols + BN - 1) / BN;
    if (s.grad && unit < blocks * a.slots) {   // the same for the whole cluster
        const int slot = unit / blocks, n0 = (unit % blocks) * BN;
        const int rank = a.rank[slot];
        int first = 0, count = 0, row = 0;
        if (rank > 0) {
            if (a.list) {
                first = a.offsets[slot];
                count = a.offsets[slot + 1] - first;
                row = a.offsets[a.slots + 2 + slot];
            } else if (slot == 0) {
                count = a.tokens;
            }
        }
        const int chunks = (count + 63) / 64, cn = max(0, (chunks - me + a.split - 1) / a.split);
        const uint32_t base = smem_u32(smem);
        float *part = reinterpret_cast<float *>(smem);   // [R][BN + 4], over the stages once they are done
        constexpr int LD = BN + 4;
        float v[MINE];
        Progress at_now = {0, 0, true};
        if (warp == READERS) {
            // lanes 0..15: the tokens of four rows of a block; asked for four blocks ahead
            constexpr int AHEAD = 4;
            int rows[AHEAD][4];
            auto ask = [&](int c, int (&r)[4]) {
                const int p = (c * a.split + me) * 64 + 4 * (lane & 15);
#pragma unroll
                for (int i = 0; i < 4; i++) r[i] = c < cn && p + i < count ? token_at(a, first + p + i) : a.tokens;
            };
#pragma unroll
            for (int u = 0; u < AHEAD; u++) ask(u, rows[u]);
            bool ok = true;
            for (int c4 = 0; c4 < cn && ok; c4 += AHEAD)
#pragma unroll
                for (int u = 0; u < AHEAD; u++) {
                    const int c = c4 + u, st = c % STAGES;
                    if (c >= cn || !ok) break;
                    const bool box = neighbours(rows[u], 4);
                    if (c >= STAGES && !warp_wait(pipe.empty + 8 * st, (uint32_t)(c / STAGES - 1) & 1u)) {
                        if (lane == 0) give_up(pipe, a.status);
                        ok = false;
                        break;
                    }
                    const uint32_t at = base + st * STAGE, bar = pipe.full + 8 * st;
                    if (lane == 0) qm::mbar_expect_tx(bar, STAGE);
                    __syncwarp();
                    if (lane >= 16 && lane < 16 + G) tma_box(at + (lane - 16) * 8192, &ta.low[1 - which], 64 * (lane - 16), row + (c * a.split + me) * 64, bar);
                    if (lane < 16) {
                        if (!box) {
#pragma unroll
                            for (int j = 0; j < NG; j++) tma_rows4(at + AB + j * 8192 + lane * 512, &ta.gather[which], n0 + 64 * j, rows[u], bar);
                        } else if ((lane & 7) == 0) {
#pragma unroll
                            for (int j = 0; j < NG; j++) tma_box(at + AB + j * 8192 + lane * 512, &ta.rows[which], n0 + 64 * j, rows[u][0], bar);
                        }
                    }
                    __syncwarp();
                    ask(c + AHEAD, rows[u]);
                }
        } else if (warp == READERS + 1) {
            if (lane == 0)
                pipe_multiply<STAGES, NACC>(pipe, at_now, base, STAGE, cn, a.status, [&](uint32_t at, int acc, bool begin) {
                    const uint64_t x = tile_desc(at + AB, 8192);
#pragma unroll
                    for (int m = 0; m < MM; m++) {
                        // (a half without a partner is taken twice; the second half of the result is not read)
                        const uint64_t l = tile_desc(at + m * 16384, 2 * m + 1 < G ? 8192 : 0);
#pragma unroll
                        for (int k = 0; k < 4; k++)   // 16 tokens = 2048 bytes = 128 descriptor units
                            tc_mma(pipe.tmem + acc * MM * BN + m * BN, l + 128 * k, x + 128 * k, tc_idesc(BN, true), !begin || k > 0);
                    }
                });
        } else {
            pipe_read<MINE, NACC>(pipe, at_now, MM * BN, (warp >> 2) * MINE, cn, a.status, v);
        }
        pipe_done(pipe);
        // row m of the accumulators is rank m % R of part m / R: the smallest part first, the others onto it
#pragma unroll
        for (int p = 2; p >= 0; p--) {
            if (p < 2) __syncthreads();
            if (warp < READERS) {
                const int c = (warp >> 2) * MINE, m = c / BN, j = c % BN;   // this warp's columns lie in one product
                const int at = m * 128 + (warp & 3) * 32 + lane - p * R;    // this lane's rank, if it holds one of this part
                if (at >= 0 && at < R) {
#pragma unroll
                    for (int i = 0; i < MINE; i += 4) {
                        float4 *q = reinterpret_cast<float4 *>(part + at * LD + j + i);
                        float4 z = p == 2 ? make_float4(0.f, 0.f, 0.f, 0.f) : *q;
                        z.x += v[i]; z.y += v[i + 1]; z.z += v[i + 2]; z.w += v[i + 3];
                        *q = z;
                    }
                }
            }
        }
        __syncthreads();
        if (a.split > 1) {
            cluster_arrive();
            cluster_wait();
        }
        // The CTAs share the columns, a thread takes four of them; neighbouring threads take neighbours of the gradient's inner
        // axis, columns of A, ranks of B.
        float *grad = s.grad + slot * s.grad_slot;
        const int quads = BN / 4 / a.split;   // of one CTA
        const bool by_col = s.grad_rank > s.grad_col;
        const bool vec = s.grad_col == 1 && ((reinterpret_cast<uintptr_t>(grad) | (uintptr_t)(s.grad_rank * 4)) & 15) == 0;
        for (int e = tid; e < R * quads; e += THREADS) {
            // (quads is a power of two)
            const int r = by_col ? e / quads : e % R, col = (me * quads + (by_col ? e & (quads - 1) : e / R)) * 4;
            if (r >= a.max_rank || n0 + col >= s.cols) continue;
            float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rank && count > 0)
                w = a.split > 1 ? peers_sum4(smem_u32(part + r * LD + col), a.split) : *reinterpret_cast<const float4 *>(part + r * LD + col);
            float *to = grad + r * s.grad_rank + (n0 + col) * s.grad_col;
            if (vec && n0 + col + 3 < s.cols) {
                *reinterpret_cast<float4 *>(to) = w;
            } else {
                to[0] = w.x;
                if (n0 + col + 1 < s.cols) to[s.grad_col] = w.y;
                if (n0 + col + 2 < s.cols) to[2 * s.grad_col] = w.z;
                if (n0 + col + 3 < s.cols) to[3 * s.grad_col] = w.w;
            }
        }
        if (a.split > 1) {
            cluster_arrive();
            cluster_wait();
        }
    }
    pipe_close(pipe, TCOLS);
}

}  // namespace

extern "C" __global__ void __launch_bounds__(SHRINK_THREADS) qm_lora_shrink_r16(const __grid_constant__ QmLoraTcArgs a) { shrink<1, false>(a); }
extern "C" __global__ void __launch_bounds__(SHRINK_THREADS) qm_lora_shrink_r32(const __grid_constant__ QmLoraTcArgs a) { shrink<2, false>(a); }
extern "C" __global__ void __launch_bounds__(SHRINK_THREADS) qm_lora_shrink_r64(const __grid_constant__ QmLoraTcArgs a) { shrink<4, false>(a); }
extern "C" __global__ void __launch_bounds__(SHRINK_THREADS) qm_lora_shrink_r128(const __grid_constant__ QmLoraTcArgs a) { shrink<8, false>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(1) * 32, 3) qm_lora_expand_r16(const __grid_constant__ QmLoraBatchArgs a) { expand<1, true, false>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(1) * 32, 3) qm_lora_expand_r16_s(const __grid_constant__ QmLoraBatchArgs a) { expand<1, false, false>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(2) * 32, 3) qm_lora_expand_r32(const __grid_constant__ QmLoraBatchArgs a) { expand<2, true, false>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(2) * 32, 3) qm_lora_expand_r32_s(const __grid_constant__ QmLoraBatchArgs a) { expand<2, false, false>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(4) * 32, 3) qm_lora_expand_r64(const __grid_constant__ QmLoraBatchArgs a) { expand<4, true, false>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(4) * 32, 3) qm_lora_expand_r64_s(const __grid_constant__ QmLoraBatchArgs a) { expand<4, false, false>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(8) * 32, 2) qm_lora_expand_r128(const __grid_constant__ QmLoraBatchArgs a) { expand<8, true, false>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(8) * 32, 2) qm_lora_expand_r128_s(const __grid_constant__ QmLoraBatchArgs a) { expand<8, false, false>(a); }
extern "C" __global__ void __launch_bounds__(SHRINK_THREADS) qm_lora_shrink_r16_m(const __grid_constant__ QmLoraTcArgs a) { shrink<1, true>(a); }
extern "C" __global__ void __launch_bounds__(SHRINK_THREADS) qm_lora_shrink_r32_m(const __grid_constant__ QmLoraTcArgs a) { shrink<2, true>(a); }
extern "C" __global__ void __launch_bounds__(SHRINK_THREADS) qm_lora_shrink_r64_m(const __grid_constant__ QmLoraTcArgs a) { shrink<4, true>(a); }
extern "C" __global__ void __launch_bounds__(SHRINK_THREADS) qm_lora_shrink_r128_m(const __grid_constant__ QmLoraTcArgs a) { shrink<8, true>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(1) * 32, 3) qm_lora_expand_r16_m(const __grid_constant__ QmLoraBatchArgs a) { expand<1, true, true>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(2) * 32, 3) qm_lora_expand_r32_m(const __grid_constant__ QmLoraBatchArgs a) { expand<2, true, true>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(4) * 32, 3) qm_lora_expand_r64_m(const __grid_constant__ QmLoraBatchArgs a) { expand<4, true, true>(a); }
extern "C" __global__ void __launch_bounds__(QM_LORA_EXPAND_WARPS(8) * 32, 2) qm_lora_expand_r128_m(const __grid_constant__ QmLoraBatchArgs a) { expand<8, true, true>(a); }
extern "C" __global__ void __launch_bounds__((QM_LORA_OUTER_READERS(1) + 2) * 32) qm_lora_outer_r16(const __grid_constant__ QmLoraTcArgs a) { outer<1>(a); }
extern "C" __global__ void __launch_bounds__((QM_LORA_OUTER_READERS(2) + 2) * 32) qm_lora_outer_r32(const __grid_constant__ QmLoraTcArgs a) { outer<2>(a); }
extern "C" __global__ void __launch_bounds__((QM_LORA_OUTER_READERS(4) + 2) * 32) qm_lora_outer_r64(const __grid_constant__ QmLoraTcArgs a) { outer<4>(a); }
extern "C" __global__ void __launch_bounds__((QM_LORA_OUTER_READERS(8) + 2) * 32) qm_lora_outer_r128(const __grid_constant__ QmLoraTcArgs a) { outer<8>(a); }
extern "C" __global__ void __launch_bounds__(256, 3) qm_lora_few_r16(const __grid_constant__ QmLoraFewArgs a) { few<1, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 3) qm_lora_few_r16_s(const __grid_constant__ QmLoraFewArgs a) { few<1, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_few_r32(const __grid_constant__ QmLoraFewArgs a) { few<2, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_few_r32_s(const __grid_constant__ QmLoraFewArgs a) { few<2, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_few_r64(const __grid_constant__ QmLoraFewArgs a) { few<4, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) qm_lora_few_r64_s(const __grid_constant__ QmLoraFewArgs a) { few<4, false>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_few_r128(const __grid_constant__ QmLoraFewArgs a) { few<8, true>(a); }
extern "C" __global__ void __launch_bounds__(256) qm_lora_few_r128_s(const __grid_constant__ QmLoraFewArgs a) { few<8, false>(a); }
