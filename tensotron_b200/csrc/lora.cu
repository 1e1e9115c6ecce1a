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

#include "lora_common.cuh"

namespace tt {
namespace lora {

namespace cg = cooperative_groups;

namespace {

constexpr int THREADS = 256;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

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
// and the 256 / (4 RP) k groups of the CTA share out the contraction index of every chunk of 64.  Chunks of x and of the
// adapter arrive through a ring of asynchronous copies, both with the contraction index contiguous, so that a 128-bit
// load of each makes two packed multiply-adds per output (sums over even and odd indices, added at the end).  The CTAs of
// a cluster cut the contraction into contiguous ranges; k groups are added through shared memory, the cluster's partial
// tiles through distributed shared memory, both in ascending order.
struct ShrinkParams {
    Groups g;
    const float* x;       // (rows, L)
    const float* w;       // KMAJ: (count, rank, L), else (count, L, rank)
    const float* scale;   // (count) or null
    float* out;           // (rows, rank)
    int rows, L, rank;
    int x_vec, w_vec;     // 128-bit copies are possible
};

template <int RP>
struct ShrinkCfg {
    static constexpr int KC = 64, LD = KC + 4, STAGES = 3;
    static constexpr int X_FLOATS = TM * LD, STAGE_FLOATS = X_FLOATS + RP * LD;
    static constexpr int SMEM_BYTES = STAGES * STAGE_FLOATS * 4;      // (the partial tiles reuse it: 4 * 256 * 16 bytes at most)
};

template <int RP, bool KMAJ>
__global__ void __launch_bounds__(THREADS) shrink_kernel(const ShrinkParams p)
{
    using C = ShrinkCfg<RP>;
    constexpr int KC = C::KC, LD = C::LD, GROUP = 4 * RP, KG = THREADS / GROUP, QPG = KC / 4 / KG;
    constexpr int XL = TM * KC / 4 / THREADS;                       // copies of x per thread and chunk
    extern __shared__ __align__(16) float smem[];
    __shared__ int row_s[TM];
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
    const int chunks = l1 > l0 ? (l1 - l0 + KC - 1) / KC : 0;
    const float* w = p.w + (tile.adapter < 0 ? 0ll : static_cast<long long>(tile.adapter) * p.rank * p.L);

    const int xc = (tid % (KC / 4)) * 4;
    const float* xsrc[XL];
#pragma unroll
    for (int i = 0; i < XL; i++) {
        const int r = row_s[tid / (KC / 4) + i * (THREADS / (KC / 4))];
        xsrc[i] = r < 0 ? nullptr : p.x + static_cast<long long>(r) * p.L + l0 + xc;
    }
    const auto issue = [&](int chunk) {
        if (chunk < chunks) {
            float* xs = smem + (chunk % C::STAGES) * C::STAGE_FLOATS;
            float* ws = xs + C::X_FLOATS;
            const int l = l0 + chunk * KC;
#pragma unroll
            for (int i = 0; i < XL; i++) {
                const int left = xsrc[i] ? l1 - l - xc : 0;
                copy4(xs + (tid / (KC / 4) + i * (THREADS / (KC / 4))) * LD + xc, left > 0 ? xsrc[i] + chunk * KC : p.x, left, p.x_vec);
            }
            if (KMAJ) {
#pragma unroll
                for (int q = tid; q < RP * KC / 4; q += THREADS) {
                    const int r = q / (KC / 4), c = (q % (KC / 4)) * 4, left = rb + r < p.rank ? l1 - l - c : 0;
                    copy4(ws + r * LD + c, left > 0 ? w + static_cast<long long>(rb + r) * p.L + l + c : p.w, left, p.w_vec);
                }
            } else {
#pragma unroll 4
                for (int q = tid; q < RP * KC; q += THREADS) {
                    const int c = q / RP, r = q % RP;
                    const bool there = l + c < l1 && rb + r < p.rank;
                    copy1(ws + r * LD + c, there ? w + static_cast<long long>(l + c) * p.rank + rb + r : p.w, there);
                }
            }
        }
        commit_copies();
    };

    const int kg = tid / GROUP, t = tid % GROUP, rg = t % 16, cgp = t / 16;
    float2 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = make_float2(0.f, 0.f);
    for (int s = 0; s < C::STAGES - 1; s++) issue(s);
    for (int chunk = 0; chunk < chunks; chunk++) {
        wait_copies<C::STAGES - 2>();
        __syncthreads();
        issue(chunk + C::STAGES - 1);
        const float* xs = smem + (chunk % C::STAGES) * C::STAGE_FLOATS;
        const float* ws = xs + C::X_FLOATS;
#pragma unroll
        for (int qq = 0; qq < QPG; qq++) {
            const int k = (kg * QPG + qq) * 4;
            float4 xv[4], wv[4];
#pragma unroll
            for (int i = 0; i < 4; i++) xv[i] = *reinterpret_cast<const float4*>(xs + (rg + 16 * i) * LD + k);
#pragma unroll
            for (int j = 0; j < 4; j++) wv[j] = *reinterpret_cast<const float4*>(ws + (cgp + RP / 4 * j) * LD + k);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __ffma2_rn(make_float2(xv[i].x, xv[i].y), make_float2(wv[j].x, wv[j].y), acc[i][j]);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __ffma2_rn(make_float2(xv[i].z, xv[i].w), make_float2(wv[j].z, wv[j].w), acc[i][j]);
        }
    }
    wait_copies<0>();
    __syncthreads();
    // partial tiles [kg][row][rank]
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) smem[(kg * TM + rg + 16 * i) * RP + cgp + RP / 4 * j] = acc[i][j].x + acc[i][j].y;
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

// 64 rows x `tiles_per` column tiles of 128; a warp owns 8 rows, a lane 4 adjacent columns of each.  Bound by the read and
// write of c, so what a step needs (the tile of c, read and written by the same thread, and up to RC ranks of the adapter)
// arrives through a two-stage ring of asynchronous copies while the step before it is computed and stored; the rows' t and
// the row numbers are read once per CTA.  More than RC ranks take several steps per column tile.
struct ExpandParams {
    Groups g;
    const float* t;       // (rows, rank)
    const float* w;       // RMAJ: (count, J, rank), else (count, rank, J)
    const float* scale;   // (count) or null
    float* c;             // (rows, J)
    int rows, J, rank, act, tiles_per;
    int w_vec, c_vec;
};

constexpr int EN = 128;

template <int RC>
struct ExpandCfg {
    static constexpr int STAGES = 2, LD = EN + 4, C_FLOATS = TM * EN, STAGE_FLOATS = C_FLOATS + RC * LD;
    static int smem_bytes(int rank) { return (STAGES * STAGE_FLOATS + TM * ((rank + RC - 1) / RC * RC)) * 4; }
};

template <int RC, bool RMAJ>
__global__ void __launch_bounds__(THREADS, 2) expand_kernel(const ExpandParams p)
{
    using C = ExpandCfg<RC>;
    extern __shared__ __align__(16) float smem[];
    __shared__ int row_s[TM];
    const Tile tile = tile_of(p.g, blockIdx.x, p.rows);
    if (!tile.valid || (tile.adapter < 0 && p.act == 0)) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rchunks = (p.rank + RC - 1) / RC, rpad = rchunks * RC;
    float* ts = smem + C::STAGES * C::STAGE_FLOATS;          // [TM][rpad], scaled
    if (tid < TM) row_s[tid] = tid < tile.rows ? (p.g.perm ? __ldg(p.g.perm + tile.first + tid) : tile.first + tid) : -1;
    __syncthreads();
    const int ct0 = blockIdx.y * p.tiles_per, ct1 = min((p.J + EN - 1) / EN, ct0 + p.tiles_per);
    const int steps = (ct1 - ct0) * rchunks;
    const float* w = p.w + static_cast<long long>(tile.adapter < 0 ? 0 : tile.adapter) * p.rank * p.J;
    float* crow[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int m = row_s[warp * 8 + i];
        crow[i] = m < 0 ? nullptr : p.c + static_cast<long long>(m) * p.J;
    }
    const auto issue = [&](int step) {
        if (step < steps) {
            const int ct = ct0 + step / rchunks, rc = step % rchunks, j0 = ct * EN, r0 = rc * RC;
            float* cs = smem + (step % C::STAGES) * C::STAGE_FLOATS;
            float* ws = cs + C::C_FLOATS;
            if (rc == 0) {                                   // (stays in its stage for this step; kept in registers for the others)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int left = crow[i] ? p.J - j0 - lane * 4 : 0;
                    copy4(cs + (warp * 8 + i) * EN + lane * 4, left > 0 ? crow[i] + j0 + lane * 4 : p.c, left, p.c_vec);
                }
            }
            if (tile.adapter >= 0) {
                if (RMAJ) {
                    // B is read along its ranks and stored rank by rank
#pragma unroll 4
                    for (int q = tid; q < EN * RC; q += THREADS) {
                        const int n = q / RC, r = q % RC;
                        const bool there = j0 + n < p.J && r0 + r < p.rank;
                        copy1(ws + r * C::LD + n, there ? w + static_cast<long long>(j0 + n) * p.rank + r0 + r : p.w, there);
                    }
                } else {
#pragma unroll
                    for (int q = tid; q < RC * (EN / 4); q += THREADS) {
                        const int r = q / (EN / 4), n = (q % (EN / 4)) * 4, left = r0 + r < p.rank ? p.J - j0 - n : 0;
                        copy4(ws + r * C::LD + n, left > 0 ? w + static_cast<long long>(r0 + r) * p.J + j0 + n : p.w, left, p.w_vec);
                    }
                }
            }
        }
        commit_copies();
    };
    issue(0);
    if (tile.adapter >= 0) {
        const float scale = p.scale ? __ldg(p.scale + tile.adapter) : 1.f;
        for (int e = tid; e < TM * rpad; e += THREADS) {
            const int r = e / rpad, c = e - r * rpad;
            ts[e] = row_s[r] >= 0 && c < p.rank ? scale * __ldg(p.t + static_cast<long long>(row_s[r]) * p.rank + c) : 0.f;
        }
    }
    float4 cv[8], acc[8];
    for (int step = 0; step < steps; step++) {
        issue(step + 1);
        wait_copies<1>();
        __syncthreads();
        const int rc = step % rchunks, j = (ct0 + step / rchunks) * EN + lane * 4, left = p.J - j;
        const float* cs = smem + (step % C::STAGES) * C::STAGE_FLOATS;
        const float* ws = cs + C::C_FLOATS;
        if (rc == 0) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                cv[i] = *reinterpret_cast<const float4*>(cs + (warp * 8 + i) * EN + lane * 4);
                acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
        if (tile.adapter >= 0) {
#pragma unroll
            for (int r = 0; r < RC; r += 4) {
                float4 wv[4];
#pragma unroll
                for (int q = 0; q < 4; q++) wv[q] = *reinterpret_cast<const float4*>(ws + (r + q) * C::LD + lane * 4);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float4 tv = *reinterpret_cast<const float4*>(ts + (warp * 8 + i) * rpad + rc * RC + r);
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
        if (rc == rchunks - 1) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (!crow[i]) continue;
                float4 v = make_float4(cv[i].x + acc[i].x, cv[i].y + acc[i].y, cv[i].z + acc[i].z, cv[i].w + acc[i].w);
                if (p.act) {
                    v.x = act_apply(v.x, p.act); v.y = act_apply(v.y, p.act);
                    v.z = act_apply(v.z, p.act); v.w = act_apply(v.w, p.act);
                }
                float* dst = crow[i] + j;
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
        __syncthreads();
    }
}

// ---- outer ----------------------------------------------------------------------------------------

// out = small^T . big over one adapter's rows: a tile of RP ranks x 128 columns.  A thread owns 8 ranks x 4 columns; the
// 4 RP threads that cover the tile once form a row group, and the row groups of the CTA share out the rows of every
// chunk of 32, which arrive through a ring of asynchronous copies.  The CTAs of a cluster cut the adapter's rows into
// contiguous ranges.  Joins as in shrink_kernel.  Two jobs in one grid: dA (rank, K) from dt and x, dB (N, rank) from t
// and g.
struct OuterJob {
    const float* small;   // (rows, rank)
    const float* big;     // (rows, C)
    float* out;           // (count, rank, C), or (count, C, rank) when col_major
    const float* scale;   // (count) or null
    int C, col_major, tiles, big_vec, small_vec;
};

struct OuterParams {
    Groups g;
    OuterJob job[2];
    int rows, rank;
};

template <int RP>
struct OuterCfg {
    static constexpr int MC = 32, CN = 128, STAGES = 3, STAGE_FLOATS = MC * CN + MC * RP;
    static constexpr int RED_FLOATS = THREADS / (4 * RP) * RP * CN;
    static constexpr int SMEM_BYTES = (STAGES * STAGE_FLOATS > RED_FLOATS ? STAGES * STAGE_FLOATS : RED_FLOATS) * 4;
};

template <int RP>
__global__ void __launch_bounds__(THREADS) outer_kernel(const OuterParams p)
{
    using C = OuterCfg<RP>;
    constexpr int MC = C::MC, CN = C::CN, GROUP = 4 * RP, MG = THREADS / GROUP;
    constexpr int BL = MC * CN / 4 / THREADS;
    extern __shared__ __align__(16) float smem[];
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
    const int chunks = m1 > m0 ? (m1 - m0 + MC - 1) / MC : 0;

    const auto issue = [&](int chunk) {
        if (chunk < chunks) {
            float* bs = smem + (chunk % C::STAGES) * C::STAGE_FLOATS;
            float* ss = bs + MC * CN;
            const int m = m0 + chunk * MC;
            const int cl = (tid % (CN / 4)) * 4;
#pragma unroll
            for (int i = 0; i < BL; i++) {
                const int r = tid / (CN / 4) + i * (THREADS / (CN / 4));
                const int left = m + r < m1 ? job.C - c0 - cl : 0;
                const long long row = left > 0 ? (p.g.perm ? __ldg(p.g.perm + first + m + r) : m + r) : 0;
                copy4(bs + r * CN + cl, left > 0 ? job.big + row * job.C + c0 + cl : job.big, left, job.big_vec);
            }
#pragma unroll
            for (int q = tid; q < MC * RP / 4; q += THREADS) {
                const int r = q / (RP / 4), c = rb + (q % (RP / 4)) * 4;
                const int left = m + r < m1 ? p.rank - c : 0;
                const long long row = left > 0 ? (p.g.perm ? __ldg(p.g.perm + first + m + r) : m + r) : 0;
                copy4(ss + q * 4, left > 0 ? job.small + row * p.rank + c : job.small, left, job.small_vec);
            }
        }
        commit_copies();
    };
    const int mg = tid / GROUP, t = tid % GROUP, cl = t % 32, rg = t / 32;   // rg: 8 ranks, cl: 4 columns
    float4 acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < C::STAGES - 1; s++) issue(s);
    for (int chunk = 0; chunk < chunks; chunk++) {
        wait_copies<C::STAGES - 2>();
        __syncthreads();
        issue(chunk + C::STAGES - 1);
        const float* bs = smem + (chunk % C::STAGES) * C::STAGE_FLOATS;
        const float* ss = bs + MC * CN;
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
    }
    wait_copies<0>();
    __syncthreads();
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
cudaError_t launch_cluster(cudaStream_t st, void (*kernel)(P), dim3 grid, int cluster, int smem, const P& p)
{
    cudaLaunchConfig_t cfg = {};
    cfg.dynamicSmemBytes = smem;
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
    p.w_vec = down && aligned16(p.w) && L % 4 == 0;
    const int tiles = g.perm ? g.max_tiles : (rows + TM - 1) / TM;
    const int rp = ad.rank <= 8 ? 8 : ad.rank <= 16 ? 16 : ad.rank <= 32 ? 32 : 64;
    const int rblocks = (ad.rank + rp - 1) / rp;
    int S = 1;
    while (S < 8 && static_cast<long long>(tiles) * rblocks * S < 3ll * num_sms && L / (2 * S) >= 64) S *= 2;
    const dim3 grid(static_cast<unsigned int>(tiles) * S, rblocks, 1);
    if (down) {
        if (rp == 8)       return launch_cluster(st, shrink_kernel<8, true>, grid, S, ShrinkCfg<8>::SMEM_BYTES, p);
        else if (rp == 16) return launch_cluster(st, shrink_kernel<16, true>, grid, S, ShrinkCfg<16>::SMEM_BYTES, p);
        else if (rp == 32) return launch_cluster(st, shrink_kernel<32, true>, grid, S, ShrinkCfg<32>::SMEM_BYTES, p);
        return launch_cluster(st, shrink_kernel<64, true>, grid, S, ShrinkCfg<64>::SMEM_BYTES, p);
    }
    if (rp == 8)       return launch_cluster(st, shrink_kernel<8, false>, grid, S, ShrinkCfg<8>::SMEM_BYTES, p);
    else if (rp == 16) return launch_cluster(st, shrink_kernel<16, false>, grid, S, ShrinkCfg<16>::SMEM_BYTES, p);
    else if (rp == 32) return launch_cluster(st, shrink_kernel<32, false>, grid, S, ShrinkCfg<32>::SMEM_BYTES, p);
    return launch_cluster(st, shrink_kernel<64, false>, grid, S, ShrinkCfg<64>::SMEM_BYTES, p);
}

cudaError_t launch_expand(cudaStream_t st, const Groups& g, const Adapters& ad, bool up, bool scaled, const float* t,
                          float* c, int rows, int J, int act, int num_sms)
{
    ExpandParams p;
    p.g = g;
    p.t = t;
    p.w = up ? ad.b : ad.a;
    p.scale = scaled ? ad.scale : nullptr;
    p.c = c;
    p.rows = rows; p.J = J; p.rank = ad.rank; p.act = act;
    p.w_vec = !up && aligned16(p.w) && J % 4 == 0;
    p.c_vec = aligned16(c) && J % 4 == 0;
    const int tiles = g.perm ? g.max_tiles : (rows + TM - 1) / TM, cols = (J + EN - 1) / EN;
    // column tiles per CTA: as many as leave four CTAs per SM
    long long per = static_cast<long long>(tiles) * cols / (4ll * num_sms);
    p.tiles_per = static_cast<int>(per < 1 ? 1 : per > 8 ? 8 : per);
    const dim3 grid(tiles, (cols + p.tiles_per - 1) / p.tiles_per, 1);
    const int rc = ad.rank <= 8 ? 8 : ad.rank <= 16 ? 16 : 32;
    if (up) {
        if (rc == 8)       expand_kernel<8, true><<<grid, THREADS, ExpandCfg<8>::smem_bytes(ad.rank), st>>>(p);
        else if (rc == 16) expand_kernel<16, true><<<grid, THREADS, ExpandCfg<16>::smem_bytes(ad.rank), st>>>(p);
        else               expand_kernel<32, true><<<grid, THREADS, ExpandCfg<32>::smem_bytes(ad.rank), st>>>(p);
    } else {
        if (rc == 8)       expand_kernel<8, false><<<grid, THREADS, ExpandCfg<8>::smem_bytes(ad.rank), st>>>(p);
        else if (rc == 16) expand_kernel<16, false><<<grid, THREADS, ExpandCfg<16>::smem_bytes(ad.rank), st>>>(p);
        else               expand_kernel<32, false><<<grid, THREADS, ExpandCfg<32>::smem_bytes(ad.rank), st>>>(p);
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
    if (da) p.job[jobs++] = OuterJob{dt, x, da, nullptr, K, 0, (K + 127) / 128, aligned16(x) && K % 4 == 0, aligned16(dt) && ad.rank % 4 == 0};
    if (db) p.job[jobs++] = OuterJob{t, grad, db, ad.scale, N, 1, (N + 127) / 128, aligned16(grad) && N % 4 == 0, aligned16(t) && ad.rank % 4 == 0};
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
    if (rp == 8)       return launch_cluster(st, outer_kernel<8>, grid, S, OuterCfg<8>::SMEM_BYTES, p);
    else if (rp == 16) return launch_cluster(st, outer_kernel<16>, grid, S, OuterCfg<16>::SMEM_BYTES, p);
    else if (rp == 32) return launch_cluster(st, outer_kernel<32>, grid, S, OuterCfg<32>::SMEM_BYTES, p);
    return launch_cluster(st, outer_kernel<64>, grid, S, OuterCfg<64>::SMEM_BYTES, p);
}

namespace {
template <typename K>
cudaError_t allow_smem(K* kernel, int bytes) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); }

template <int RP>
cudaError_t init_rank()
{
    cudaError_t e;
    if ((e = allow_smem(shrink_kernel<RP, true>, ShrinkCfg<RP>::SMEM_BYTES)) != cudaSuccess) return e;
    if ((e = allow_smem(shrink_kernel<RP, false>, ShrinkCfg<RP>::SMEM_BYTES)) != cudaSuccess) return e;
    return allow_smem(outer_kernel<RP>, OuterCfg<RP>::SMEM_BYTES);
}

template <int RC>
cudaError_t init_expand()
{
    const int bytes = ExpandCfg<RC>::smem_bytes(RC == 32 ? MAX_RANK : RC);
    const cudaError_t e = allow_smem(expand_kernel<RC, true>, bytes);
    return e != cudaSuccess ? e : allow_smem(expand_kernel<RC, false>, bytes);
}
}  // namespace

cudaError_t init_tiled()
{
    cudaError_t e;
    if ((e = init_rank<8>()) != cudaSuccess || (e = init_rank<16>()) != cudaSuccess || (e = init_rank<32>()) != cudaSuccess ||
        (e = init_rank<64>()) != cudaSuccess || (e = init_expand<8>()) != cudaSuccess || (e = init_expand<16>()) != cudaSuccess)
        return e;
    return init_expand<32>();
}

}  // namespace lora
}  // namespace tt
