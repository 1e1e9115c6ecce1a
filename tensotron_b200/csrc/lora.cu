// Low-rank adapters beside a shared projection.  Row m of a call has adapter e_m (or none); with A (rank, K), B (N, rank)
// and the scale s of its adapter
//     forward    t = A x            y  = act(y + s B t)
//     backward   dt = s B^T g       dx = dx + A^T dt       dA = sum_m dt x^T       dB = s sum_m g t^T
// All arithmetic is float32 fused multiply-adds, sums in an order that depends on the shapes and the grouping only.
//
// Rows are grouped by adapter first (group_kernel), so that a tile of 64 rows meets one adapter: its A and B are then
// read once per tile from L2, and the four products become three tiled kernels:
//     shrink_kernel   (rows x L) . (L x rank): a long contraction into a narrow output
//     expand_kernel   (rows x rank) . (rank x J), added to what the output holds
//     outer_kernel    (rank x rows) . (rows x C): contracts over the rows of one adapter
#include "lora.h"

#include <cooperative_groups.h>
#include <stdint.h>

#include "ptx.cuh"

namespace tt {
namespace lora {

namespace cg = cooperative_groups;

namespace {

constexpr int THREADS = 256;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

__device__ __forceinline__ float act_apply(float v, int act)
{
    if (act == 1) return v > 0.f ? v : 0.f;
    if (act == 2) return tanhf(v);
    return v;
}

// Four consecutive floats at p, of which the first `n` exist (the others read as 0).
__device__ __forceinline__ float4 load4(const float* p, int n, bool vec)
{
    if (vec && n >= 4) return __ldg(reinterpret_cast<const float4*>(p));
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (n > 0) v.x = __ldg(p);
    if (n > 1) v.y = __ldg(p + 1);
    if (n > 2) v.z = __ldg(p + 2);
    if (n > 3) v.w = __ldg(p + 3);
    return v;
}

// ---- grouping of the rows -----------------------------------------------------------------------

// One CTA per group (adapters 0 .. count-1, then the rows without one).  A CTA counts the rows of all lower groups and,
// warp by warp over contiguous row ranges, its own; the range counts give every warp its place, and a second walk
// writes the row indices.  No atomics on the data: ascending row order within a group, whatever the timing.  The
// last CTA to finish lists the tiles.
__global__ void __launch_bounds__(THREADS)
group_kernel(Groups g, const int* __restrict__ row_adapter, int rows, int count, unsigned int* ticket, unsigned int* status)
{
    constexpr int WARPS = THREADS / 32;
    __shared__ int below_s[WARPS], own_s[WARPS], carry_s[WARPS];
    __shared__ unsigned int last;
    const int e = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = ((rows + WARPS - 1) / WARPS + 31) & ~31;
    const int r0 = warp * per, r1 = min(rows, r0 + per);
    int below = 0, own = 0;
    bool bad = false;
    for (int r = r0 + lane; r < r1; r += 32) {
        int k = __ldg(row_adapter + r);
        if (k < 0 || k >= count) {
            bad |= k != -1;
            k = count;
        }
        below += k < e;
        own += k == e;
    }
    if (bad && status) atomicCAS(status, 0u, static_cast<unsigned int>(DEV_BAD_ADAPTER));
    below = __reduce_add_sync(0xffffffffu, below);
    own = __reduce_add_sync(0xffffffffu, own);
    if (lane == 0) { below_s[warp] = below; own_s[warp] = own; }
    __syncthreads();
    int base = 0, mine = 0, total = 0;
    for (int w = 0; w < WARPS; w++) {
        base += below_s[w];
        if (w < warp) mine += own_s[w];
        total += own_s[w];
    }
    int at = base + mine;
    if (total > 0) {
        for (int r = r0; r < r1; r += 32) {
            int k = r + lane < r1 ? __ldg(row_adapter + r + lane) : count + 1;
            if (r + lane < r1 && (k < 0 || k >= count)) k = count;
            const unsigned int hit = __ballot_sync(0xffffffffu, k == e);
            if (k == e) g.perm[at + __popc(hit & ((1u << lane) - 1u))] = r + lane;
            at += __popc(hit);
        }
    }
    if (threadIdx.x == 0) {
        g.offset[e] = base;
        if (e == count) g.offset[count + 1] = rows;
        __threadfence();
        last = atomicAdd(ticket, 1u) == gridDim.x - 1 ? 1u : 0u;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    // tile list: an exclusive scan of ceil(rows / TM) over the groups, THREADS groups at a time
    int first_tile = 0;
    for (int g0 = 0; g0 <= count; g0 += THREADS) {
        const int k = g0 + threadIdx.x;
        int lo = 0, n = 0;
        if (k <= count) {
            lo = __ldcg(g.offset + k);
            n = __ldcg(g.offset + k + 1) - lo;
        }
        const int tiles = (n + TM - 1) / TM;
        int inc = tiles;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        __syncthreads();
        if (lane == 31) carry_s[warp] = inc;
        __syncthreads();
        int before = first_tile, all = 0;
        for (int w = 0; w < WARPS; w++) {
            if (w < warp) before += carry_s[w];
            all += carry_s[w];
        }
        int tile = before + inc - tiles;
        for (int i = 0; i < tiles; i++, tile++) {
            g.tile_adapter[tile] = k < count ? k : -1;
            g.tile_first[tile] = lo + i * TM;
            g.tile_rows[tile] = min(TM, n - i * TM);
        }
        first_tile += all;
    }
    if (threadIdx.x == 0) {
        *g.n_tiles = first_tile;
        *ticket = 0u;
    }
}

struct Tile {
    int adapter, first, rows;
    bool valid;
};

__device__ __forceinline__ Tile tile_of(const Groups& g, int i, int rows)
{
    Tile t;
    if (g.perm) {
        t.valid = i < __ldg(g.n_tiles);
        if (!t.valid) return t;
        t.adapter = __ldg(g.tile_adapter + i);
        t.first = __ldg(g.tile_first + i);
        t.rows = __ldg(g.tile_rows + i);
    } else {
        t.adapter = 0;
        t.first = i * TM;
        t.rows = min(TM, rows - t.first);
        t.valid = t.rows > 0;
    }
    return t;
}

// ---- shrink ---------------------------------------------------------------------------------------

// A tile of 64 rows x RP ranks.  A thread owns 4 x 4 outputs; the 4 RP threads that cover the tile once form a k group,
// and the 256 / (4 RP) k groups of the CTA share out the contraction index of every chunk of 32.  The CTAs of a cluster
// cut the contraction into contiguous ranges; k groups are added through shared memory, the cluster's partial tiles
// through distributed shared memory, both in ascending order.
struct ShrinkParams {
    Groups g;
    const float* x;       // (rows, L)
    const float* w;       // KMAJ: (count, rank, L), else (count, L, rank)
    const float* scale;   // (count) or null
    float* out;           // (rows, rank)
    int rows, L, rank;
    int x_vec, w_vec;     // 128-bit loads are possible
};

template <int RP, bool KMAJ>
__global__ void __launch_bounds__(THREADS) shrink_kernel(const ShrinkParams p)
{
    constexpr int KC = 32, LD = KC + 4, GROUP = 4 * RP, KG = THREADS / GROUP, QPG = KC / 4 / KG;
    constexpr int X_FLOATS = TM * LD, W_FLOATS = KMAJ ? RP * LD : KC * (RP + 4);
    constexpr int RED_FLOATS = KG * TM * RP;
    constexpr int SMEM = X_FLOATS + W_FLOATS > RED_FLOATS ? X_FLOATS + W_FLOATS : RED_FLOATS;
    constexpr int XL = TM * KC / 4 / THREADS;                       // float4 of x per thread and chunk
    constexpr int WL = (RP * KC / 4 + THREADS - 1) / THREADS;
    __shared__ __align__(16) float smem[SMEM];
    __shared__ int row_s[TM];
    float* xs = smem;
    float* ws = smem + X_FLOATS;
    cg::cluster_group cluster = cg::this_cluster();
    const int S = static_cast<int>(cluster.num_blocks()), split = static_cast<int>(cluster.block_rank());
    const int tid = threadIdx.x;
    const int rb = blockIdx.y * RP;                                  // first rank of this block of ranks
    const Tile tile = tile_of(p.g, blockIdx.x / S, p.rows);
    if (!tile.valid) return;                                         // (the whole cluster)
    if (tid < TM) row_s[tid] = tid < tile.rows ? (p.g.perm ? __ldg(p.g.perm + tile.first + tid) : tile.first + tid) : -1;
    __syncthreads();
    const int span = ((p.L + S - 1) / S + KC - 1) / KC * KC;
    const int l0 = split * span, l1 = tile.adapter < 0 ? 0 : min(p.L, l0 + span);
    const float* w = p.w + (tile.adapter < 0 ? 0ll : static_cast<long long>(tile.adapter) * p.rank * p.L);

    float4 xr[XL], wr[WL];
    const auto fetch = [&](int l) {
#pragma unroll
        for (int i = 0; i < XL; i++) {
            const int q = tid + i * THREADS, r = q / (KC / 4), c = l + (q % (KC / 4)) * 4;
            xr[i] = row_s[r] < 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                                 : load4(p.x + static_cast<long long>(row_s[r]) * p.L + c, l1 - c, p.x_vec);
        }
#pragma unroll
        for (int i = 0; i < WL; i++) {
            const int q = tid + i * THREADS;
            wr[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (q < RP * KC / 4) {
                if (KMAJ) {
                    const int r = q / (KC / 4), c = l + (q % (KC / 4)) * 4;
                    if (rb + r < p.rank) wr[i] = load4(w + static_cast<long long>(rb + r) * p.L + c, l1 - c, p.w_vec);
                } else {
                    const int c = l + q / (RP / 4), r = rb + (q % (RP / 4)) * 4;
                    if (c < l1) wr[i] = load4(w + static_cast<long long>(c) * p.rank + r, p.rank - r, p.w_vec);
                }
            }
        }
    };

    const int kg = tid / GROUP, t = tid % GROUP, rg = t % 16, cgp = t / 16;
    float acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = 0.f;
    if (l0 < l1) fetch(l0);
    for (int l = l0; l < l1; l += KC) {
#pragma unroll
        for (int i = 0; i < XL; i++) {
            const int q = tid + i * THREADS;
            *reinterpret_cast<float4*>(xs + (q / (KC / 4)) * LD + (q % (KC / 4)) * 4) = xr[i];
        }
#pragma unroll
        for (int i = 0; i < WL; i++) {
            const int q = tid + i * THREADS;
            if (q < RP * KC / 4) {
                if (KMAJ) *reinterpret_cast<float4*>(ws + (q / (KC / 4)) * LD + (q % (KC / 4)) * 4) = wr[i];
                else      *reinterpret_cast<float4*>(ws + (q / (RP / 4)) * (RP + 4) + (q % (RP / 4)) * 4) = wr[i];
            }
        }
        __syncthreads();
        if (l + KC < l1) fetch(l + KC);
#pragma unroll
        for (int qq = 0; qq < QPG; qq++) {
            const int k = (kg * QPG + qq) * 4;
            float xv[4][4], wv[4][4];                    // [row][k], [rank][k]
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<float4*>(xv[i]) = *reinterpret_cast<const float4*>(xs + (rg + 16 * i) * LD + k);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (KMAJ) {
                    *reinterpret_cast<float4*>(wv[j]) = *reinterpret_cast<const float4*>(ws + (cgp + RP / 4 * j) * LD + k);
                } else {
                    const float4 v = *reinterpret_cast<const float4*>(ws + (k + j) * (RP + 4) + cgp * 4);
                    wv[0][j] = v.x; wv[1][j] = v.y; wv[2][j] = v.z; wv[3][j] = v.w;
                }
            }
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[i][j] = fmaf(xv[i][kk], wv[j][kk], acc[i][j]);
        }
        __syncthreads();
    }
    // partial tiles [kg][row][rank]
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            smem[(kg * TM + rg + 16 * i) * RP + (KMAJ ? cgp + RP / 4 * j : cgp * 4 + j)] = acc[i][j];
    __syncthreads();
    for (int e = tid; e < TM * RP && KG > 1; e += THREADS) {
        float s = smem[e];
#pragma unroll
        for (int q = 1; q < KG; q++) s += smem[q * TM * RP + e];
        smem[e] = s;
    }
    const float scale = p.scale && tile.adapter >= 0 ? __ldg(p.scale + tile.adapter) : 1.f;
    if (S > 1) cluster.sync(); else __syncthreads();
    const int rows_per = TM / S;
    for (int e = tid; e < rows_per * RP; e += THREADS) {
        const int r = split * rows_per + e / RP, c = e % RP;
        if (row_s[r] < 0 || rb + c >= p.rank) continue;
        float s = S > 1 ? *cluster.map_shared_rank(smem + r * RP + c, 0) : smem[r * RP + c];
        for (int q = 1; q < S; q++) s += *cluster.map_shared_rank(smem + r * RP + c, q);
        p.out[static_cast<long long>(row_s[r]) * p.rank + rb + c] = scale * s;
    }
    if (S > 1) cluster.sync();      // nobody leaves while its partial tile may still be read
}

// ---- expand ---------------------------------------------------------------------------------------

// A tile of 64 rows x 128 columns; a warp owns 8 rows, a lane 4 adjacent columns of each.  Ranks are taken 32 at a
// time.  Bound by the read and write of c; its values are fetched before the products are formed.
struct ExpandParams {
    Groups g;
    const float* t;       // (rows, rank)
    const float* w;       // RMAJ: (count, J, rank), else (count, rank, J)
    const float* scale;   // (count) or null
    float* c;             // (rows, J)
    int rows, J, rank, act;
    int w_vec, c_vec;
};

constexpr int EN = 128;

template <int RC, bool RMAJ>
__global__ void __launch_bounds__(THREADS) expand_kernel(const ExpandParams p)
{
    __shared__ __align__(16) float ts[TM][RC];
    __shared__ __align__(16) float ws[RC][EN + 4];
    __shared__ int row_s[TM];
    const Tile tile = tile_of(p.g, blockIdx.x, p.rows);
    if (!tile.valid || (tile.adapter < 0 && p.act == 0)) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid < TM) row_s[tid] = tid < tile.rows ? (p.g.perm ? __ldg(p.g.perm + tile.first + tid) : tile.first + tid) : -1;
    __syncthreads();
    const int j0 = blockIdx.y * EN, j = j0 + lane * 4, left = p.J - j;
    float4 cv[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int m = row_s[warp * 8 + i];
        cv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (m >= 0) {
            const float* src = p.c + static_cast<long long>(m) * p.J + j;
            if (p.c_vec && left >= 4) {
                cv[i] = *reinterpret_cast<const float4*>(src);
            } else {
                if (left > 0) cv[i].x = src[0];
                if (left > 1) cv[i].y = src[1];
                if (left > 2) cv[i].z = src[2];
                if (left > 3) cv[i].w = src[3];
            }
        }
    }
    float4 acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (tile.adapter >= 0) {
        const float* w = p.w + static_cast<long long>(tile.adapter) * p.rank * p.J;
        const float scale = p.scale ? __ldg(p.scale + tile.adapter) : 1.f;
        for (int r0 = 0; r0 < p.rank; r0 += RC) {
            const int rn = min(RC, p.rank - r0);
            if (r0) __syncthreads();
            for (int e = tid; e < TM * RC; e += THREADS) {
                const int r = e / RC, c = e % RC;
                ts[r][c] = row_s[r] >= 0 && c < rn ? scale * __ldg(p.t + static_cast<long long>(row_s[r]) * p.rank + r0 + c) : 0.f;
            }
            if (RMAJ) {
                for (int e = tid; e < EN * (RC / 4); e += THREADS) {
                    const int n = e / (RC / 4), r = (e % (RC / 4)) * 4;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (j0 + n < p.J) v = load4(w + static_cast<long long>(j0 + n) * p.rank + r0 + r, rn - r, p.w_vec);
                    ws[r][n] = v.x; ws[r + 1][n] = v.y; ws[r + 2][n] = v.z; ws[r + 3][n] = v.w;
                }
            } else {
                for (int e = tid; e < RC * (EN / 4); e += THREADS) {
                    const int r = e / (EN / 4), n = (e % (EN / 4)) * 4;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (r < rn) v = load4(w + static_cast<long long>(r0 + r) * p.J + j0 + n, p.J - j0 - n, p.w_vec);
                    *reinterpret_cast<float4*>(&ws[r][n]) = v;
                }
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < RC; r += 4) {
                float4 wv[4];
#pragma unroll
                for (int q = 0; q < 4; q++) wv[q] = *reinterpret_cast<const float4*>(&ws[r + q][lane * 4]);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float4 tv = *reinterpret_cast<const float4*>(&ts[warp * 8 + i][r]);
                    const float t4[4] = {tv.x, tv.y, tv.z, tv.w};
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        acc[i].x = fmaf(t4[q], wv[q].x, acc[i].x);
                        acc[i].y = fmaf(t4[q], wv[q].y, acc[i].y);
                        acc[i].z = fmaf(t4[q], wv[q].z, acc[i].z);
                        acc[i].w = fmaf(t4[q], wv[q].w, acc[i].w);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int m = row_s[warp * 8 + i];
        if (m < 0) continue;
        float4 v = make_float4(cv[i].x + acc[i].x, cv[i].y + acc[i].y, cv[i].z + acc[i].z, cv[i].w + acc[i].w);
        if (p.act) {
            v.x = act_apply(v.x, p.act); v.y = act_apply(v.y, p.act);
            v.z = act_apply(v.z, p.act); v.w = act_apply(v.w, p.act);
        }
        float* dst = p.c + static_cast<long long>(m) * p.J + j;
        if (p.c_vec && left >= 4) {
            *reinterpret_cast<float4*>(dst) = v;
        } else {
            if (left > 0) dst[0] = v.x;
            if (left > 1) dst[1] = v.y;
            if (left > 2) dst[2] = v.z;
            if (left > 3) dst[3] = v.w;
        }
    }
}

// ---- outer ----------------------------------------------------------------------------------------

// out = small^T . big over one adapter's rows: a tile of RP ranks x 128 columns.  A thread owns 8 ranks x 4 columns; the
// 4 RP threads that cover the tile once form a row group, and the row groups of the CTA share out the rows of every
// chunk of 32.  The CTAs of a cluster cut the adapter's rows into contiguous ranges.  Joins as in shrink_kernel.  Two
// jobs in one grid: dA (rank, K) from dt and x, dB (N, rank) from t and g.
struct OuterJob {
    const float* small;   // (rows, rank)
    const float* big;     // (rows, C)
    float* out;           // (count, rank, C), or (count, C, rank) when col_major
    const float* scale;   // (count) or null
    int C, col_major, tiles, big_vec;
};

struct OuterParams {
    Groups g;
    OuterJob job[2];
    int rows, rank;
};

template <int RP>
__global__ void __launch_bounds__(THREADS) outer_kernel(const OuterParams p)
{
    constexpr int MC = 32, CN = 128, GROUP = 4 * RP, MG = THREADS / GROUP;
    constexpr int RED_FLOATS = MG * RP * CN, IN_FLOATS = MC * CN + MC * RP;
    constexpr int SMEM = RED_FLOATS > IN_FLOATS ? RED_FLOATS : IN_FLOATS;
    constexpr int BL = MC * CN / 4 / THREADS, SL = (MC * RP + THREADS - 1) / THREADS;
    __shared__ __align__(16) float smem[SMEM];
    float* bs = smem;
    float* ss = smem + MC * CN;
    cg::cluster_group cluster = cg::this_cluster();
    const int S = static_cast<int>(cluster.num_blocks()), split = static_cast<int>(cluster.block_rank());
    const int tid = threadIdx.x, e = blockIdx.y, rb = blockIdx.z * RP;
    int ct = blockIdx.x / S;
    const OuterJob& job = p.job[ct < p.job[0].tiles ? 0 : 1];
    if (ct >= p.job[0].tiles) ct -= p.job[0].tiles;
    const int c0 = ct * CN;
    int first = 0, n = p.rows;
    if (p.g.perm) {
        first = __ldg(p.g.offset + e);
        n = __ldg(p.g.offset + e + 1) - first;
    } else if (e > 0) {
        n = 0;
    }
    const int span = ((n + S - 1) / S + MC - 1) / MC * MC;
    const int m0 = split * span, m1 = min(n, m0 + span);

    float4 br[BL];
    float sr[SL];
    const auto row_of = [&](int m) { return p.g.perm ? __ldg(p.g.perm + first + m) : m; };
    const auto fetch = [&](int m) {
#pragma unroll
        for (int i = 0; i < BL; i++) {
            const int q = tid + i * THREADS, r = m + q / (CN / 4), c = c0 + (q % (CN / 4)) * 4;
            br[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < m1) br[i] = load4(job.big + static_cast<long long>(row_of(r)) * job.C + c, job.C - c, job.big_vec);
        }
#pragma unroll
        for (int i = 0; i < SL; i++) {
            const int q = tid + i * THREADS, r = m + q / RP, c = rb + q % RP;
            sr[i] = 0.f;
            if (q < MC * RP && r < m1 && c < p.rank) sr[i] = __ldg(job.small + static_cast<long long>(row_of(r)) * p.rank + c);
        }
    };
    const int mg = tid / GROUP, t = tid % GROUP, cl = t % 32, rg = t / 32;   // rg: 8 ranks, cl: 4 columns
    float4 acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (m0 < m1) fetch(m0);
    for (int m = m0; m < m1; m += MC) {
#pragma unroll
        for (int i = 0; i < BL; i++) *reinterpret_cast<float4*>(bs + (tid + i * THREADS) * 4) = br[i];
#pragma unroll
        for (int i = 0; i < SL; i++)
            if (tid + i * THREADS < MC * RP) ss[tid + i * THREADS] = sr[i];
        __syncthreads();
        if (m + MC < m1) fetch(m + MC);
#pragma unroll 4
        for (int r = mg; r < MC; r += MG) {
            const float4 bv = *reinterpret_cast<const float4*>(bs + r * CN + cl * 4);
            float sv[8];
            *reinterpret_cast<float4*>(sv) = *reinterpret_cast<const float4*>(ss + r * RP + rg * 8);
            *reinterpret_cast<float4*>(sv + 4) = *reinterpret_cast<const float4*>(ss + r * RP + rg * 8 + 4);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                acc[i].x = fmaf(sv[i], bv.x, acc[i].x);
                acc[i].y = fmaf(sv[i], bv.y, acc[i].y);
                acc[i].z = fmaf(sv[i], bv.z, acc[i].z);
                acc[i].w = fmaf(sv[i], bv.w, acc[i].w);
            }
        }
        __syncthreads();
    }
    // partial tiles [mg][rank][column]
#pragma unroll
    for (int i = 0; i < 8; i++) *reinterpret_cast<float4*>(smem + (mg * RP + rg * 8 + i) * CN + cl * 4) = acc[i];
    __syncthreads();
    if (MG > 1) {
        for (int q = tid; q < RP * CN; q += THREADS) {
            float s = smem[q];
#pragma unroll
            for (int k = 1; k < MG; k++) s += smem[k * RP * CN + q];
            smem[q] = s;
        }
    }
    const float scale = job.scale ? __ldg(job.scale + e) : 1.f;
    float* out = job.out + static_cast<long long>(e) * p.rank * job.C;
    if (S > 1) cluster.sync(); else __syncthreads();
    const int per = RP * CN / S;
    for (int q = tid; q < per; q += THREADS) {
        const int k = split * per + q;
        // neighbouring threads write neighbouring addresses in either layout
        const int r = job.col_major ? k % RP : k / CN, c = job.col_major ? k / RP : k % CN;
        if (rb + r >= p.rank || c0 + c >= job.C) continue;
        float s = S > 1 ? *cluster.map_shared_rank(smem + r * CN + c, 0) : smem[r * CN + c];
        for (int o = 1; o < S; o++) s += *cluster.map_shared_rank(smem + r * CN + c, o);
        out[job.col_major ? static_cast<long long>(c0 + c) * p.rank + rb + r : static_cast<long long>(rb + r) * job.C + c0 + c] = scale * s;
    }
    if (S > 1) cluster.sync();
}

template <typename P>
cudaError_t launch_cluster(cudaStream_t st, void (*kernel)(P), dim3 grid, int cluster, const P& p)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned int>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

size_t up256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// Tiles a grouping can have: every group ends with at most one partial tile.
int tile_bound(int rows, int adapters)
{
    const int groups = rows < adapters + 1 ? rows : adapters + 1;
    return rows / TM + groups;
}

}  // namespace

size_t groups_bytes(int rows, int adapters)
{
    return up256(sizeof(int) * static_cast<size_t>(rows)) + up256(sizeof(int) * (static_cast<size_t>(adapters) + 3)) +
           3 * up256(sizeof(int) * static_cast<size_t>(tile_bound(rows, adapters)));
}

Groups groups_layout(void* mem, int rows, int adapters)
{
    Groups g;
    uint8_t* at = static_cast<uint8_t*>(mem);
    g.max_tiles = tile_bound(rows, adapters);
    const size_t t = up256(sizeof(int) * static_cast<size_t>(g.max_tiles));
    g.perm = reinterpret_cast<int*>(at);
    at += up256(sizeof(int) * static_cast<size_t>(rows));
    g.offset = reinterpret_cast<int*>(at);
    g.n_tiles = g.offset + adapters + 2;
    at += up256(sizeof(int) * (static_cast<size_t>(adapters) + 3));
    g.tile_adapter = reinterpret_cast<int*>(at);
    g.tile_first = reinterpret_cast<int*>(at + t);
    g.tile_rows = reinterpret_cast<int*>(at + 2 * t);
    return g;
}

cudaError_t launch_group(cudaStream_t st, const Groups& g, const int* row_adapter, int rows, int adapters,
                         unsigned int* ticket, unsigned int* status)
{
    group_kernel<<<adapters + 1, THREADS, 0, st>>>(g, row_adapter, rows, adapters, ticket, status);
    return cudaGetLastError();
}

cudaError_t launch_shrink(cudaStream_t st, const Groups& g, const Adapters& ad, bool down, bool scaled, const float* x,
                          float* out, int rows, int L, int num_sms)
{
    ShrinkParams p;
    p.g = g;
    p.x = x;
    p.w = down ? ad.a : ad.b;
    p.scale = scaled ? ad.scale : nullptr;
    p.out = out;
    p.rows = rows; p.L = L; p.rank = ad.rank;
    p.x_vec = aligned16(x) && L % 4 == 0;
    p.w_vec = aligned16(p.w) && (down ? L : ad.rank) % 4 == 0;
    const int tiles = g.perm ? g.max_tiles : (rows + TM - 1) / TM;
    const int rp = ad.rank <= 8 ? 8 : ad.rank <= 16 ? 16 : ad.rank <= 32 ? 32 : 64;
    const int rblocks = (ad.rank + rp - 1) / rp;
    int S = 1;
    while (S < 8 && static_cast<long long>(tiles) * rblocks * S < 3ll * num_sms && L / (2 * S) >= 64) S *= 2;
    const dim3 grid(static_cast<unsigned int>(tiles) * S, rblocks, 1);
    if (down) {
        if (rp == 8)       return launch_cluster(st, shrink_kernel<8, true>, grid, S, p);
        else if (rp == 16) return launch_cluster(st, shrink_kernel<16, true>, grid, S, p);
        else if (rp == 32) return launch_cluster(st, shrink_kernel<32, true>, grid, S, p);
        return launch_cluster(st, shrink_kernel<64, true>, grid, S, p);
    }
    if (rp == 8)       return launch_cluster(st, shrink_kernel<8, false>, grid, S, p);
    else if (rp == 16) return launch_cluster(st, shrink_kernel<16, false>, grid, S, p);
    else if (rp == 32) return launch_cluster(st, shrink_kernel<32, false>, grid, S, p);
    return launch_cluster(st, shrink_kernel<64, false>, grid, S, p);
}

cudaError_t launch_expand(cudaStream_t st, const Groups& g, const Adapters& ad, bool up, bool scaled, const float* t,
                          float* c, int rows, int J, int act)
{
    ExpandParams p;
    p.g = g;
    p.t = t;
    p.w = up ? ad.b : ad.a;
    p.scale = scaled ? ad.scale : nullptr;
    p.c = c;
    p.rows = rows; p.J = J; p.rank = ad.rank; p.act = act;
    p.w_vec = aligned16(p.w) && (up ? ad.rank : J) % 4 == 0;
    p.c_vec = aligned16(c) && J % 4 == 0;
    const int tiles = g.perm ? g.max_tiles : (rows + TM - 1) / TM;
    const dim3 grid(tiles, (J + EN - 1) / EN, 1);
    if (grid.y > 65535u) return cudaErrorInvalidValue;
    const int rc = ad.rank <= 8 ? 8 : ad.rank <= 16 ? 16 : 32;
    if (up) {
        if (rc == 8)       expand_kernel<8, true><<<grid, THREADS, 0, st>>>(p);
        else if (rc == 16) expand_kernel<16, true><<<grid, THREADS, 0, st>>>(p);
        else               expand_kernel<32, true><<<grid, THREADS, 0, st>>>(p);
    } else {
        if (rc == 8)       expand_kernel<8, false><<<grid, THREADS, 0, st>>>(p);
        else if (rc == 16) expand_kernel<16, false><<<grid, THREADS, 0, st>>>(p);
        else               expand_kernel<32, false><<<grid, THREADS, 0, st>>>(p);
    }
    return cudaGetLastError();
}

cudaError_t launch_outer(cudaStream_t st, const Groups& g, const Adapters& ad, const float* dt, const float* x, float* da,
                         const float* grad, const float* t, float* db, int rows, int N, int K, int num_sms)
{
    OuterParams p;
    p.g = g;
    p.rows = rows;
    p.rank = ad.rank;
    int jobs = 0;
    p.job[0].tiles = p.job[1].tiles = 0;
    if (da) p.job[jobs++] = OuterJob{dt, x, da, nullptr, K, 0, (K + 127) / 128, aligned16(x) && K % 4 == 0};
    if (db) p.job[jobs++] = OuterJob{t, grad, db, ad.scale, N, 1, (N + 127) / 128, aligned16(grad) && N % 4 == 0};
    if (jobs == 0) return cudaSuccess;
    if (jobs == 1) { p.job[1] = p.job[0]; p.job[1].tiles = 0; }
    const int rp = ad.rank <= 8 ? 8 : ad.rank <= 16 ? 16 : ad.rank <= 32 ? 32 : 64;
    const int rblocks = (ad.rank + rp - 1) / rp;
    const int tiles = p.job[0].tiles + p.job[1].tiles;
    const int groups = g.perm ? ad.count : 1;
    int S = 1;
    while (S < 8 && static_cast<long long>(tiles) * rblocks * groups * S < 3ll * num_sms && rows / (2 * S * groups) >= 32) S *= 2;
    // (without a grouping the adapters behind the first have no rows: their CTAs store zeros)
    const dim3 grid(static_cast<unsigned int>(tiles) * S, ad.count, rblocks);
    if (rp == 8)       return launch_cluster(st, outer_kernel<8>, grid, S, p);
    else if (rp == 16) return launch_cluster(st, outer_kernel<16>, grid, S, p);
    else if (rp == 32) return launch_cluster(st, outer_kernel<32>, grid, S, p);
    return launch_cluster(st, outer_kernel<64>, grid, S, p);
}

}  // namespace lora
}  // namespace tt
