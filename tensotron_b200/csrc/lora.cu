// Low-rank adapters beside a shared projection.  Row m of a call has adapter e_m (or none); with A (rank, K), B (N, rank)
// and the scale s of its adapter
//     forward    t = A x            y  = act(y + s B t)
//     backward   dt = s B^T g       dx = dx + A^T dt       dA = sum_m dt x^T       dB = s sum_m g t^T
// All arithmetic is float32 fused multiply-adds, sums in an order that depends on the shapes and the grouping only.
//
// Rows are grouped by adapter first (group_kernel), so that a tile of 64 rows meets one adapter: its A and B are then
// read once per tile from L2, and the four products become three tiled kernels:
//     shrink_kernel   (rows x L) . (L x rank): a long contraction into a narrow output; 8192 x 4096 at rank 16: 41-49 us for
//                     134 MB and 1.07 GFLOP (20.5 and 14.5 us at their rates)
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

constexpr int THREADS = 256, GROUP_THREADS = 1024;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The launches of a call overlap: each lets the next one begin (let_next_begin) once the launches in front of it are known
// to be complete, and waits (wait_for_previous) where it first reads what the one in front of it writes, or at its end.  So
// at any point behind a wait, and at the start of a launch that was let begin, everything but the launch directly in
// front is complete.
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// At the end of a kernel whose CTAs need not have waited: one of them does, so that this launch is not complete before the
// one in front of it, and the others leave their SM.
__device__ __forceinline__ void finish()
{
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) wait_for_previous();
}

// ---- grouping of the rows -----------------------------------------------------------------------

// One CTA per group (adapters 0 .. count-1, then the rows without one).  A CTA counts the rows of all lower groups and,
// warp by warp over contiguous row ranges, its own; the range counts give every warp its place, and a second walk
// writes the row indices.  No atomics: ascending row order within a group, whatever the timing.  Bound by latency: 8192 rows,
// 8 adapters 4.6 us, 333 rows 3.1.
__global__ void __launch_bounds__(GROUP_THREADS)
group_kernel(Groups g, const int* __restrict__ row_adapter, int rows, int count, unsigned int* status)
{
    constexpr int WARPS = GROUP_THREADS / 32, AHEAD = 4;
    __shared__ int below_s[WARPS], own_s[WARPS];
    let_next_begin();
    const int e = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = ((rows + WARPS - 1) / WARPS + 31) & ~31;
    const int r0 = warp * per, r1 = min(rows, r0 + per);
    int below = 0, own = 0;
    bool bad = false;
#pragma unroll 8
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
        for (int r = r0; r < r1; r += 32 * AHEAD) {
            int k[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int at_row = r + 32 * i + lane;
                k[i] = at_row < r1 ? __ldg(row_adapter + at_row) : e + 1;                 // (not this group's)
                if (at_row < r1 && (k[i] < 0 || k[i] >= count)) k[i] = count;
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const unsigned int hit = __ballot_sync(0xffffffffu, k[i] == e);
                if (k[i] == e) g.perm[at + __popc(hit & ((1u << lane) - 1u))] = r + 32 * i + lane;
                at += __popc(hit);
            }
        }
    }
    if (threadIdx.x == 0) {
        g.offset[e] = base;
        if (e == count) g.offset[count + 1] = rows;
    }
}

struct Tile {
    int adapter, first, rows;     // adapter -1: the rows without one
    bool valid;
};

// All threads of the CTA: tile `i` of the call.  The tiles follow the groups, ceil(rows / TM) for each, so every CTA finds its
// own by a scan over the groups' sizes (a list made by the grouping would cost it a second round through memory).
__device__ __forceinline__ Tile tile_of(const Groups& g, int i, int rows)
{
    Tile t;
    if (!g.perm) {
        t.adapter = 0;
        t.first = i * TM;
        t.rows = min(TM, rows - t.first);
        t.valid = t.rows > 0;
        return t;
    }
    __shared__ int carry_s[THREADS / 32];
    __shared__ Tile found;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) found.valid = false;
    int before = 0;
    for (int g0 = 0; g0 <= g.count && before <= i; g0 += THREADS) {
        const int k = g0 + threadIdx.x;
        int lo = 0, n = 0;
        if (k <= g.count) {
            lo = __ldcg(g.offset + k);
            n = __ldcg(g.offset + k + 1) - lo;
        }
        const int tiles = (n + TM - 1) / TM;
        int inc = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) carry_s[warp] = inc;
        __syncthreads();
        int first = before + inc - tiles, all = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 32; w++) {
            if (w < warp) first += carry_s[w];
            all += carry_s[w];
        }
        if (i >= first && i < first + tiles) {
            found.adapter = k < g.count ? k : -1;
            found.first = lo + (i - first) * TM;
            found.rows = min(TM, n - (i - first) * TM);
            found.valid = true;
        }
        before += all;
        __syncthreads();
    }
    return found;
}

// Rows of a tile as their numbers in the call, -1 behind the last one.
__device__ __forceinline__ void tile_row_numbers(const Groups& g, const Tile& tile, int* row_s)
{
    if (threadIdx.x < TM)
        row_s[threadIdx.x] = static_cast<int>(threadIdx.x) < tile.rows ? (g.perm ? __ldcg(g.perm + tile.first + threadIdx.x) : tile.first + static_cast<int>(threadIdx.x)) : -1;
}

// The tiled kernels take their operands through rings of stages filled by asynchronous copies, of 16 bytes where every row
// starts on such a boundary and is a multiple of 16 bytes long (VEC), else of 4.  Every thread copies the same places of
// every stage, so that a copy costs an addition and the instruction itself.  (Bulk copies, one per row of a stage, were
// tried: about 45 cycles each per SM whatever their length, 8192 x 4096 rows in 104 us against 55.)  Rows behind the last one
// of a tile repeat its first (their outputs are not stored); the rings start on 128-byte boundaries (16 bytes beside one, the
// copies of a 512-byte row took an extra pass each: expand_kernel 62 us against 54); what lies behind the last index of a contraction is 0 or is
// not looked at.

// ---- shrink ---------------------------------------------------------------------------------------

// A tile of 64 rows x RP ranks.  The contraction index goes in slices of 16, dealt to the warps in turn; a warp covers all
// 64 rows and RW (8 or 16) ranks of its slices, 4 rows x RW / 2 ranks per lane, and keeps them in a ring of its own, so that warps with
// different slices never wait for one another (with a ring shared by the CTA and a barrier per 128 k: 59 us for 8192 x 4096
// rows at rank 16, against 51 us).  Ranks beyond 16 take 2 or 4 warps per slice, which share its rows and a barrier.
// The adapter's part of a slice is kept with the ranks contiguous: a packed multiply-add serves two of them.  KMAJ: in memory its
// contraction index is contiguous, it is copied in pieces of 4 bytes.  The CTAs of a cluster cut the contraction into
// contiguous ranges; slices are added through shared memory, the cluster's partial tiles through distributed shared
// memory, both in ascending order.
struct ShrinkParams {
    Groups g;
    const float* x;       // (rows, L)
    const float* w;       // KMAJ: (count, rank, L), else (count, L, rank)
    const float* scale;   // (count) or null
    float* out;           // (rows, rank)
    int rows, L, rank;
};

template <int RP, bool KMAJ>
struct ShrinkCfg {
    static constexpr int KW = 16, LD = KW + 4, RW = RP < 16 ? RP : 16, RT = RW / 2;
    static constexpr int RB = RP / RW, KS = THREADS / 32 / RB;                  // warps per slice, slices at a time
    // (rows of 16 ranks, 16 floats apart, would put the pieces of a K-major copy on two banks)
    static constexpr int X_FLOATS = TM * LD, PITCH = KMAJ ? RW + 4 : RW, W_FLOATS = KW * PITCH, STAGE_FLOATS = X_FLOATS + RB * W_FLOATS;
    static constexpr int STAGES = RB == 1 ? 2 : 3;
    static constexpr int RED_FLOATS = KS * TM * RP, RING_FLOATS = KS * STAGES * STAGE_FLOATS;
    static constexpr int SMEM_BYTES = (RING_FLOATS > RED_FLOATS ? RING_FLOATS : RED_FLOATS) * 4;
};

template <int RP, bool KMAJ, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) shrink_kernel(const __grid_constant__ ShrinkParams p)
{
    using C = ShrinkCfg<RP, KMAJ>;
    constexpr int KW = C::KW, LD = C::LD, STAGES = C::STAGES, RW = C::RW, RT = C::RT, RB = C::RB, KS = C::KS, Q = KW / 4;
    extern __shared__ __align__(128) float smem[];
    __shared__ int row_s[TM];
    cg::cluster_group cluster = cg::this_cluster();
    const int S = static_cast<int>(cluster.num_blocks()), split = static_cast<int>(cluster.block_rank());
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, ks = warp / RB, wr = warp % RB;
    const int rb = blockIdx.y * RP;                                  // first rank of this block of ranks
    wait_for_previous();
    let_next_begin();
    const Tile tile = tile_of(p.g, blockIdx.x / S, p.rows);
    if (!tile.valid) return;                                         // (the whole cluster)
    tile_row_numbers(p.g, tile, row_s);
    __syncthreads();
    constexpr int ROUND = KW * KS;                                   // contraction indices that the CTA takes at a time
    const int span = ((p.L + S - 1) / S + ROUND - 1) / ROUND * ROUND;
    const int l0 = split * span + ks * KW, l1 = tile.adapter < 0 ? 0 : min(p.L, split * span + span);
    const int chunks = l1 > l0 ? (l1 - l0 + ROUND - 1) / ROUND : 0;  // of this warp
    const float* w = p.w + (tile.adapter < 0 ? 0ll : static_cast<long long>(tile.adapter) * p.rank * p.L);
    const int r0 = rb + wr * RW, wn = min(RW, p.rank - r0);          // this warp's ranks (wn <= 0: none)
    float* ring = smem + ks * STAGES * C::STAGE_FLOATS;

    // VEC: this lane's places of a stage
    constexpr int XN = TM * Q / 32 / RB, WN = KMAJ ? 1 : RW * Q / 32;
    const int c4 = (lane % Q) * 4, xr = wr * (TM / RB) + lane / Q;
    constexpr int XSTEP = 32 / Q;
    int xat[XN], wat[WN];                      // (element offsets: int32 reaches every element of x and of one adapter)
    bool wok[WN];
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < XN; i++) {
            const int r = row_s[xr + i * XSTEP];
            xat[i] = (r < 0 ? row_s[0] : r) * p.L + l0 + c4;
        }
#pragma unroll
        for (int i = 0; i < WN; i++) {
            const int q = lane + 32 * i;
            if constexpr (KMAJ) {
                wat[0] = (r0 + lane / KW) * p.L + l0 + lane % KW;
            } else {
                wok[i] = (q % (RW / 4)) * 4 < wn;
                wat[i] = (l0 + q / (RW / 4)) * p.rank + r0 + (q % (RW / 4)) * 4;
            }
        }
    }
    const auto issue = [&](int chunk) {
        if (chunk < chunks) {
            float* xs = ring + (chunk % STAGES) * C::STAGE_FLOATS;
            float* ws = xs + C::X_FLOATS + wr * C::W_FLOATS;
            const int at = chunk * ROUND, l = l0 + at, kn = min(KW, l1 - l);
            if constexpr (VEC) {
                if (c4 < kn) {
#pragma unroll
                    for (int i = 0; i < XN; i++) copy16(xs + (xr + i * XSTEP) * LD + c4, p.x + xat[i] + at);
                }
                if constexpr (KMAJ) {
                    if (lane % KW < kn) {
                        const float* src = w + wat[0] + at;
                        float* dst = ws + (lane % KW) * C::PITCH + lane / KW;
#pragma unroll
                        for (int i = 0; i < RW * KW / 32; i++)
                            if (lane / KW + i * (32 / KW) < wn) copy1(dst + i * (32 / KW), src + i * (32 / KW) * p.L, true);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < WN; i++) {
                        const int q = lane + 32 * i;
                        if (wok[i] && q / (RW / 4) < kn) copy16(ws + q * 4, w + wat[i] + at * p.rank);
                    }
                }
            } else {
                for (int q = lane + 32 * wr; q < TM * KW; q += 32 * RB) {
                    const int r = q / KW, c = q % KW;
                    const bool there = c < kn && row_s[r] >= 0;
                    copy1(xs + r * LD + c, there ? p.x + static_cast<long long>(row_s[r]) * p.L + l + c : p.x, there);
                }
                for (int q = lane; q < RW * KW; q += 32) {
                    const int r = KMAJ ? q / KW : q % RW, c = KMAJ ? q % KW : q / RW;
                    const bool there = c < kn && r < wn;
                    copy1(ws + c * C::PITCH + r,
                          there ? w + (KMAJ ? static_cast<long long>(r0 + r) * p.L + l + c : static_cast<long long>(l + c) * p.rank + r0 + r) : p.w, there);
                }
            }
        }
        commit_copies();
    };
    // the warps of one slice
    const auto meet = [&]() {
        if constexpr (RB == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + ks), "n"(32 * RB) : "memory");
    };

    const int rg = lane % 16, cgp = lane / 16;
    constexpr int NA = RT / 2;
    float2 acc[4][NA];                         // [row][pair of ranks]
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < NA; j++) acc[i][j] = make_float2(0.f, 0.f);
    for (int s = 0; s < STAGES - 1; s++) issue(s);
    for (int done = 0; done < chunks; done++) {
        if constexpr (STAGES > 2) {
            wait_copies<STAGES - 2>();
            meet();
            issue(done + STAGES - 1);
        } else {
            // (two stages: the other one was read in the previous step, by the same warp)
            __syncwarp();
            issue(done + 1);
            wait_copies<1>();
            __syncwarp();
        }
        const float* xs = ring + (done % STAGES) * C::STAGE_FLOATS;
        const float* ws = xs + C::X_FLOATS + wr * C::W_FLOATS;
        const int kn = min(KW, l1 - l0 - done * ROUND);
#pragma unroll
        for (int k = 0; k < KW; k += 4) {
            if (k >= kn) break;
            float4 xv[4];
#pragma unroll
            for (int i = 0; i < 4; i++) xv[i] = *reinterpret_cast<const float4*>(xs + (rg + 16 * i) * LD + k);
#pragma unroll
            for (int kk = 0; kk < 4; kk++) {
#pragma unroll
                for (int j = 0; j < RT / 4; j++) {
                    const float4 wv = *reinterpret_cast<const float4*>(ws + (k + kk) * C::PITCH + cgp * RT + 4 * j);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float xk = kk == 0 ? xv[i].x : kk == 1 ? xv[i].y : kk == 2 ? xv[i].z : xv[i].w;
                        acc[i][2 * j] = __ffma2_rn(make_float2(xk, xk), make_float2(wv.x, wv.y), acc[i][2 * j]);
                        acc[i][2 * j + 1] = __ffma2_rn(make_float2(xk, xk), make_float2(wv.z, wv.w), acc[i][2 * j + 1]);
                    }
                }
            }
        }
    }
    wait_copies<0>();
    __syncthreads();
    // partial tiles [slice][row][rank]
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < RT; j++)
            smem[(ks * TM + rg + 16 * i) * RP + wr * RW + cgp * RT + j] = j & 1 ? acc[i][j / 2].y : acc[i][j / 2].x;
    __syncthreads();
    for (int e = tid; e < TM * RP; e += THREADS) {
        float s = smem[e];
#pragma unroll
        for (int q = 1; q < KS; q++) s += smem[q * TM * RP + e];
        smem[e] = s;
    }
    const float scale = p.scale && tile.adapter >= 0 ? __ldg(p.scale + tile.adapter) : 1.f;
    if (S > 1) cluster.sync(); else __syncthreads();
    for (int e = split * THREADS + tid; e < TM * RP; e += S * THREADS) {
        const int r = e / RP, c = e % RP;
        if (row_s[r] < 0 || rb + c >= p.rank) continue;
        float s = S > 1 ? *cluster.map_shared_rank(smem + r * RP + c, 0) : smem[r * RP + c];
        for (int q = 1; q < S; q++) s += *cluster.map_shared_rank(smem + r * RP + c, q);
        p.out[static_cast<long long>(row_s[r]) * p.rank + rb + c] = scale * s;
    }
    if (S > 1) cluster.sync();      // nobody leaves while its partial tile may still be read
}

// ---- expand ---------------------------------------------------------------------------------------

// 64 rows x `tiles_per` column tiles of 128; a warp owns 8 rows, a lane 4 adjacent columns of each.  Bound by the read and
// write of c: a step (up to RC ranks of one column tile) asks for its part of c and for the adapter's ranks of the next
// step, then computes, then adds c, which the same thread asked for and stores, so that c takes one buffer and no
// barrier.  The rows' t are read once per CTA and kept rank by rank: a packed multiply-add takes two rows.
// 8192 x 4096 at rank 16: 53 us for 268 MB (41 us at the copy rate); what it waits for is shared memory at 24 warps per SM.
struct ExpandParams {
    Groups g;
    const float* t;       // (rows, rank)
    const float* w;       // RMAJ: (count, J, rank), else (count, rank, J)
    const float* scale;   // (count) or null
    float* c;             // (rows, J)
    int rows, J, rank, act, tiles_per;
    int wait_first;       // the launch in front writes t, or c
};

constexpr int EN = 128;

template <int RC>
struct ExpandCfg {
    static constexpr int LD = EN + 4, C_FLOATS = TM * EN, W_FLOATS = RC * LD;
    static int smem_bytes(int rank) { return (C_FLOATS + 2 * W_FLOATS + TM * rank) * 4; }
};

template <int RC, bool RMAJ, bool VEC>
__global__ void __launch_bounds__(THREADS, 3) expand_kernel(const __grid_constant__ ExpandParams p)
{
    using C = ExpandCfg<RC>;
    extern __shared__ __align__(128) float smem[];
    __shared__ int row_s[TM];
    const Tile tile = tile_of(p.g, blockIdx.x, p.rows);
    if (p.wait_first) wait_for_previous();
    if (!tile.valid || (tile.adapter < 0 && p.act == 0)) {
        finish();
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool with = tile.adapter >= 0;
    const int rchunks = with ? (p.rank + RC - 1) / RC : 1;
    float* cs = smem;                                      // [TM][EN]
    float* wring = smem + C::C_FLOATS;                     // [2][RC][LD]
    float* ts = wring + 2 * C::W_FLOATS;                   // [rank][TM], scaled
    tile_row_numbers(p.g, tile, row_s);
    __syncthreads();
    const int ct0 = blockIdx.y * p.tiles_per, ct1 = min((p.J + EN - 1) / EN, ct0 + p.tiles_per);
    const int steps = (ct1 - ct0) * rchunks;
    const float* w = p.w + static_cast<long long>(with ? tile.adapter : 0) * p.rank * p.J;

    const auto issue_c = [&](int ct) {
        const int j0 = (ct0 + ct) * EN, jn = min(EN, p.J - j0);
        if constexpr (VEC) {
            if (lane * 4 < jn) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int m = row_s[warp * 8 + i];       // (int32 offsets reach every element of c)
                    copy16(cs + (warp * 8 + i) * EN + lane * 4, p.c + ((m < 0 ? row_s[0] : m) * p.J + j0 + lane * 4));
                }
            }
        } else {
            for (int i = 0; i < 8; i++) {
                const int m = row_s[warp * 8 + i];
                copy4(cs + (warp * 8 + i) * EN + lane * 4, m >= 0 && lane * 4 < jn ? p.c + static_cast<long long>(m) * p.J + j0 + lane * 4 : p.c,
                      m >= 0 ? jn - lane * 4 : 0, false);
            }
        }
    };
    const auto issue_w = [&](int step) {
        if (step < steps && with) {
            const int ct = step / rchunks, rc = step - ct * rchunks, j0 = (ct0 + ct) * EN, r0 = rc * RC;
            const int jn = min(EN, p.J - j0), rn = min(RC, p.rank - r0);
            float* ws = wring + (step & 1) * C::W_FLOATS;
            if constexpr (!RMAJ) {
                if constexpr (VEC) {
                    if (lane * 4 < jn) {
#pragma unroll
                        for (int i = 0; i < RC / 8; i++)
                            if (warp + 8 * i < rn)
                                copy16(ws + (warp + 8 * i) * C::LD + lane * 4, w + static_cast<long long>(r0 + warp + 8 * i) * p.J + j0 + lane * 4);
                    }
                } else {
                    for (int q = tid; q < rn * EN; q += THREADS) {
                        const int r = q / EN, n = q % EN;
                        copy1(ws + r * C::LD + n, n < jn ? w + static_cast<long long>(r0 + r) * p.J + j0 + n : p.w, n < jn);
                    }
                }
            }
            if constexpr (RMAJ) {
                // B is read along its ranks and stored rank by rank
                constexpr int NS = THREADS / RC;
                const int r = tid % RC, n0 = tid / RC;
                const float* src = w + static_cast<long long>(j0 + n0) * p.rank + r0 + r;
                float* dst = ws + r * C::LD + n0;
                const long long hop = static_cast<long long>(NS) * p.rank;
                const int last = r < rn ? jn : 0;
#pragma unroll 8
                for (int n = n0; n < EN; n += NS, src += hop, dst += NS) copy1(dst, n < last ? src : p.w, n < last);
            }
        }
        commit_copies();
    };
    issue_w(0);
    if (with) {
        const float scale = p.scale ? __ldg(p.scale + tile.adapter) : 1.f;
        for (int e = tid; e < TM * p.rank; e += THREADS) {
            const int r = e / p.rank, c = e - r * p.rank;
            ts[c * TM + r] = row_s[r] >= 0 ? scale * __ldcg(p.t + static_cast<long long>(row_s[r]) * p.rank + c) : 0.f;
        }
    }
    float2 acc[4][4];                                      // [pair of rows][column]
    for (int step = 0; step < steps; step++) {
        const int ct = step / rchunks, rc = step - ct * rchunks;
        wait_copies<0>();                                  // this step's ranks
        __syncthreads();
        if (rc == 0) issue_c(ct);
        commit_copies();
        issue_w(step + 1);
        const float* ws = wring + (step & 1) * C::W_FLOATS + lane * 4;
        if (rc == 0) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = make_float2(0.f, 0.f);
        }
        if (with) {
            const int rn = min(RC, p.rank - rc * RC);
            const float* tp = ts + rc * RC * TM + warp * 8;
#pragma unroll 4
            for (int r = 0; r < rn; r++) {
                const float4 wv = *reinterpret_cast<const float4*>(ws + r * C::LD);
                const float4 t0 = *reinterpret_cast<const float4*>(tp + r * TM);
                const float4 t1 = *reinterpret_cast<const float4*>(tp + r * TM + 4);
                const float2 tv[4] = {make_float2(t0.x, t0.y), make_float2(t0.z, t0.w), make_float2(t1.x, t1.y), make_float2(t1.z, t1.w)};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    acc[i][0] = __ffma2_rn(tv[i], make_float2(wv.x, wv.x), acc[i][0]);
                    acc[i][1] = __ffma2_rn(tv[i], make_float2(wv.y, wv.y), acc[i][1]);
                    acc[i][2] = __ffma2_rn(tv[i], make_float2(wv.z, wv.z), acc[i][2]);
                    acc[i][3] = __ffma2_rn(tv[i], make_float2(wv.w, wv.w), acc[i][3]);
                }
            }
        }
        if (rc < rchunks - 1) continue;
        wait_copies<1>();                                  // c (the ranks of the next step may still be under way)
        const int j = (ct0 + ct) * EN + lane * 4, left = p.J - j;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int m = row_s[warp * 8 + i];
            if (m < 0 || left <= 0) continue;
            float4 v = *reinterpret_cast<const float4*>(cs + (warp * 8 + i) * EN + lane * 4);
            v.x += i & 1 ? acc[i / 2][0].y : acc[i / 2][0].x;
            v.y += i & 1 ? acc[i / 2][1].y : acc[i / 2][1].x;
            v.z += i & 1 ? acc[i / 2][2].y : acc[i / 2][2].x;
            v.w += i & 1 ? acc[i / 2][3].y : acc[i / 2][3].x;
            if (p.act) {
                v.x = act_apply(v.x, p.act); v.y = act_apply(v.y, p.act);
                v.z = act_apply(v.z, p.act); v.w = act_apply(v.w, p.act);
            }
            float* dst = p.c + static_cast<long long>(m) * p.J + j;
            if (VEC) {
                *reinterpret_cast<float4*>(dst) = v;
            } else {
                dst[0] = v.x;
                if (left > 1) dst[1] = v.y;
                if (left > 2) dst[2] = v.z;
                if (left > 3) dst[3] = v.w;
            }
        }
    }
    wait_copies<0>();
    finish();
}

// ---- outer ----------------------------------------------------------------------------------------

// out = small^T . big over one adapter's rows: a tile of RP ranks x 128 columns.  A thread owns RT (8, or 16) ranks x 4
// columns, a packed multiply-add serves two ranks; the 32 RP / RT threads that cover the tile once form a row group, and the
// row groups of the CTA share out the rows of every chunk of 64.  The CTAs of a cluster cut the adapter's rows into
// contiguous ranges.  Joins as in shrink_kernel.  Two jobs in one grid: dA (rank, K) from dt and x, dB (N, rank) from t
// and g.  8192 rows, both of 4096 columns, rank 16: 70 us for 268 MB and 2.1 GFLOP (41 and 29 us at their rates), half of the
// issue slots busy.
struct OuterJob {
    const float* small;   // (rows, rank)
    const float* big;     // (rows, C)
    float* out;           // (count, rank, C), or (count, C, rank) when col_major
    const float* scale;   // (count) or null
    int C, col_major, tiles;
    int wait_first;       // the launch in front writes `small` (or nobody else waits for it)
};

struct OuterParams {
    Groups g;
    OuterJob job[2];
    int rows, rank;
};

template <int RP>
struct OuterCfg {
    static constexpr int MC = 64, CN = 128, STAGES = 2, STAGE_FLOATS = MC * CN + MC * RP;
    static constexpr int RT = RP < 16 ? RP : 16, GROUP = 32 * (RP / RT), MG = THREADS / GROUP;
    static constexpr int RED_FLOATS = MG * RP * CN;
    static constexpr int SMEM_BYTES = (STAGES * STAGE_FLOATS > RED_FLOATS ? STAGES * STAGE_FLOATS : RED_FLOATS) * 4;
};

template <int RP, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) outer_kernel(const __grid_constant__ OuterParams p)
{
    using C = OuterCfg<RP>;
    constexpr int MC = C::MC, CN = C::CN, STAGES = C::STAGES, RT = C::RT, GROUP = C::GROUP, MG = C::MG;
    extern __shared__ __align__(128) float smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int S = static_cast<int>(cluster.num_blocks()), split = static_cast<int>(cluster.block_rank());
    const int tid = threadIdx.x, e = blockIdx.y, rb = blockIdx.z * RP;
    int ct = blockIdx.x / S;
    const OuterJob& job = p.job[ct < p.job[0].tiles ? 0 : 1];
    if (ct >= p.job[0].tiles) ct -= p.job[0].tiles;
    if (job.wait_first) wait_for_previous();
    let_next_begin();
    const int c0 = ct * CN, cn = min(CN, job.C - c0), rn = min(RP, p.rank - rb);
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

    // VEC: this thread's places of a stage, and the rows of the next fill (a grouping's are looked up a fill ahead)
    constexpr int BN = MC * CN / 4 / THREADS, Q = RP / 4, SN = (MC * Q + THREADS - 1) / THREADS;
    const int c4 = (tid % 32) * 4, br = tid / 32, s4 = (tid % Q) * 4, sr = tid / Q;
    int brow[BN], srow[SN];
    const auto look_up = [&](int chunk) {
        const int m = m0 + chunk * MC;
#pragma unroll
        for (int i = 0; i < BN; i++) brow[i] = p.g.perm ? __ldg(p.g.perm + first + min(m + br + 8 * i, m1 - 1)) : min(m + br + 8 * i, m1 - 1);
#pragma unroll
        for (int i = 0; i < SN; i++) {
            const int r = min(m + sr + i * (THREADS / Q), m1 - 1);
            srow[i] = p.g.perm ? __ldg(p.g.perm + first + r) : r;
        }
    };
    const auto issue = [&](int chunk) {
        if (chunk < chunks) {
            float* bs = smem + (chunk % STAGES) * C::STAGE_FLOATS;
            float* ss = bs + MC * CN;
            const int m = m0 + chunk * MC, mn = min(MC, m1 - m);
            if constexpr (VEC) {
                if (c4 < cn) {
#pragma unroll
                    for (int i = 0; i < BN; i++) copy16(bs + (br + 8 * i) * CN + c4, job.big + static_cast<long long>(brow[i]) * job.C + c0 + c4);
                }
                if (s4 < rn && (MC * Q >= THREADS || sr < MC)) {
#pragma unroll
                    for (int i = 0; i < SN; i++)
                        copy16(ss + (sr + i * (THREADS / Q)) * RP + s4, job.small + static_cast<long long>(srow[i]) * p.rank + rb + s4);
                }
                if (chunk + 1 < chunks) look_up(chunk + 1);
            } else {
                for (int q = tid; q < mn * CN; q += THREADS) {
                    const int r = q / CN, c = q % CN;
                    const long long row = p.g.perm ? __ldg(p.g.perm + first + m + r) : m + r;
                    copy1(bs + q, c < cn ? job.big + row * job.C + c0 + c : job.big, c < cn);
                }
                for (int q = tid; q < mn * RP; q += THREADS) {
                    const int r = q / RP, c = q % RP;
                    const long long row = p.g.perm ? __ldg(p.g.perm + first + m + r) : m + r;
                    copy1(ss + q, c < rn ? job.small + row * p.rank + rb + c : job.small, c < rn);
                }
            }
        }
        commit_copies();
    };
    if (VEC && chunks > 0) look_up(0);
    const int mg = tid / GROUP, t = tid % GROUP, cl = t % 32, rg = t / 32;   // rg: RT ranks, cl: 4 columns
    float2 acc[RT / 2][4];                                                   // [rank pair][column]
#pragma unroll
    for (int i = 0; i < RT / 2; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = make_float2(0.f, 0.f);
    for (int s = 0; s < STAGES - 1; s++) issue(s);
    for (int done = 0; done < chunks; done++) {
        wait_copies<STAGES - 2>();
        __syncthreads();
        issue(done + STAGES - 1);
        const float* bs = smem + (done % STAGES) * C::STAGE_FLOATS + cl * 4;
        const float* ss = smem + (done % STAGES) * C::STAGE_FLOATS + MC * CN + rg * RT;
        const int mn = min(MC, m1 - m0 - done * MC);
#pragma unroll 2
        for (int r = mg; r < mn; r += MG) {
            const float4 bv = *reinterpret_cast<const float4*>(bs + r * CN);
#pragma unroll
            for (int i = 0; i < RT / 4; i++) {
                const float4 sv = *reinterpret_cast<const float4*>(ss + r * RP + 4 * i);
                const float2 s0 = make_float2(sv.x, sv.y), s1 = make_float2(sv.z, sv.w);
                acc[2 * i][0] = __ffma2_rn(s0, make_float2(bv.x, bv.x), acc[2 * i][0]);
                acc[2 * i][1] = __ffma2_rn(s0, make_float2(bv.y, bv.y), acc[2 * i][1]);
                acc[2 * i][2] = __ffma2_rn(s0, make_float2(bv.z, bv.z), acc[2 * i][2]);
                acc[2 * i][3] = __ffma2_rn(s0, make_float2(bv.w, bv.w), acc[2 * i][3]);
                acc[2 * i + 1][0] = __ffma2_rn(s1, make_float2(bv.x, bv.x), acc[2 * i + 1][0]);
                acc[2 * i + 1][1] = __ffma2_rn(s1, make_float2(bv.y, bv.y), acc[2 * i + 1][1]);
                acc[2 * i + 1][2] = __ffma2_rn(s1, make_float2(bv.z, bv.z), acc[2 * i + 1][2]);
                acc[2 * i + 1][3] = __ffma2_rn(s1, make_float2(bv.w, bv.w), acc[2 * i + 1][3]);
            }
        }
    }
    wait_copies<0>();
    __syncthreads();
    // partial tiles [mg][rank][column]
#pragma unroll
    for (int i = 0; i < RT / 2; i++) {
        float* dst = smem + (mg * RP + rg * RT + 2 * i) * CN + cl * 4;
        *reinterpret_cast<float4*>(dst) = make_float4(acc[i][0].x, acc[i][1].x, acc[i][2].x, acc[i][3].x);
        *reinterpret_cast<float4*>(dst + CN) = make_float4(acc[i][0].y, acc[i][1].y, acc[i][2].y, acc[i][3].y);
    }
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
    for (int k = split * THREADS + tid; k < RP * CN; k += S * THREADS) {
        // neighbouring threads write neighbouring addresses in either layout
        const int r = job.col_major ? k % RP : k / CN, c = job.col_major ? k / RP : k % CN;
        if (r >= rn || c >= cn) continue;
        float s = S > 1 ? *cluster.map_shared_rank(smem + r * CN + c, 0) : smem[r * CN + c];
        for (int o = 1; o < S; o++) s += *cluster.map_shared_rank(smem + r * CN + c, o);
        out[job.col_major ? static_cast<long long>(c0 + c) * p.rank + rb + r : static_cast<long long>(rb + r) * job.C + c0 + c] = scale * s;
    }
    if (S > 1) cluster.sync();
    finish();
}

// `early`: the launch in front of this one is one of these kernels (it lets this one begin once all its CTAs run).
template <typename P>
cudaError_t launch_cluster(cudaStream_t st, void (*kernel)(P), dim3 grid, int cluster, int smem, bool early, const P& p)
{
    cudaLaunchConfig_t cfg = {};
    cfg.dynamicSmemBytes = smem;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned int>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = early ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

size_t up256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// Tiles a grouping can have: every group ends with at most one partial tile.
int tile_bound(int rows, int adapters)
{
    const int groups = rows < adapters + 1 ? rows : adapters + 1;
    return rows / TM + groups;
}

// CTAs of a cluster: as many as let all CTAs be resident at once, `per_sm` on each SM, with at least `least` of the
// `longest` contraction for each.
int cluster_size(long long ctas, int longest, int least, int per_sm, int num_sms)
{
    int S = 1;
    while (S < 8 && ctas * (S + 1) <= static_cast<long long>(per_sm) * num_sms && longest / (S + 1) >= least) S++;
    return S;
}

template <int RP, bool KMAJ>
cudaError_t launch_shrink_t(cudaStream_t st, const ShrinkParams& p, int tiles, bool vec, bool early, int num_sms)
{
    const int rblocks = (p.rank + RP - 1) / RP;
    const int S = cluster_size(static_cast<long long>(tiles) * rblocks, p.L, 128, 2, num_sms);
    const dim3 grid(static_cast<unsigned int>(tiles) * S, rblocks, 1);
    const int smem = ShrinkCfg<RP, KMAJ>::SMEM_BYTES;
    return vec ? launch_cluster(st, shrink_kernel<RP, KMAJ, true>, grid, S, smem, early, p)
               : launch_cluster(st, shrink_kernel<RP, KMAJ, false>, grid, S, smem, early, p);
}

template <int RC, bool RMAJ>
cudaError_t launch_expand_t(cudaStream_t st, const ExpandParams& p, dim3 grid, bool vec, bool early)
{
    const int smem = ExpandCfg<RC>::smem_bytes(p.rank);
    return vec ? launch_cluster(st, expand_kernel<RC, RMAJ, true>, grid, 1, smem, early, p)
               : launch_cluster(st, expand_kernel<RC, RMAJ, false>, grid, 1, smem, early, p);
}

template <int RP>
cudaError_t launch_outer_t(cudaStream_t st, const OuterParams& p, int groups, int count, bool vec, bool early, int num_sms)
{
    const int tiles = p.job[0].tiles + p.job[1].tiles, rblocks = (p.rank + RP - 1) / RP;
    const int S = cluster_size(static_cast<long long>(tiles) * rblocks * groups, p.rows / groups, OuterCfg<RP>::MC, 2, num_sms);
    // (without a grouping the adapters behind the first have no rows: their CTAs store zeros)
    const dim3 grid(static_cast<unsigned int>(tiles) * S, count, rblocks);
    return vec ? launch_cluster(st, outer_kernel<RP, true>, grid, S, OuterCfg<RP>::SMEM_BYTES, early, p)
               : launch_cluster(st, outer_kernel<RP, false>, grid, S, OuterCfg<RP>::SMEM_BYTES, early, p);
}

template <typename K>
cudaError_t allow_smem(K* kernel, int bytes) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); }

template <int RP, bool VEC>
cudaError_t init_rank()
{
    cudaError_t e;
    if ((e = allow_smem(shrink_kernel<RP, true, VEC>, ShrinkCfg<RP, true>::SMEM_BYTES)) != cudaSuccess) return e;
    if ((e = allow_smem(shrink_kernel<RP, false, VEC>, ShrinkCfg<RP, false>::SMEM_BYTES)) != cudaSuccess) return e;
    return allow_smem(outer_kernel<RP, VEC>, OuterCfg<RP>::SMEM_BYTES);
}

template <int RC, bool VEC>
cudaError_t init_expand()
{
    const int bytes = ExpandCfg<RC>::smem_bytes(RC == 32 ? MAX_RANK : RC);
    const cudaError_t e = allow_smem(expand_kernel<RC, true, VEC>, bytes);
    return e != cudaSuccess ? e : allow_smem(expand_kernel<RC, false, VEC>, bytes);
}

template <bool VEC>
cudaError_t init_vec()
{
    cudaError_t e;
    if ((e = init_rank<8, VEC>()) != cudaSuccess || (e = init_rank<16, VEC>()) != cudaSuccess || (e = init_rank<32, VEC>()) != cudaSuccess ||
        (e = init_rank<64, VEC>()) != cudaSuccess || (e = init_expand<8, VEC>()) != cudaSuccess || (e = init_expand<16, VEC>()) != cudaSuccess)
        return e;
    return init_expand<32, VEC>();
}

}  // namespace

size_t groups_bytes(int rows, int adapters)
{
    return up256(sizeof(int) * static_cast<size_t>(rows)) + up256(sizeof(int) * (static_cast<size_t>(adapters) + 2));
}

Groups groups_layout(void* mem, int rows, int adapters)
{
    Groups g;
    uint8_t* at = static_cast<uint8_t*>(mem);
    g.max_tiles = tile_bound(rows, adapters);
    g.count = adapters;
    g.perm = reinterpret_cast<int*>(at);
    g.offset = reinterpret_cast<int*>(at + up256(sizeof(int) * static_cast<size_t>(rows)));
    return g;
}

cudaError_t launch_group(cudaStream_t st, const Groups& g, const int* row_adapter, int rows, int adapters,
                         unsigned int* status)
{
    group_kernel<<<adapters + 1, GROUP_THREADS, 0, st>>>(g, row_adapter, rows, adapters, status);
    return cudaGetLastError();
}

cudaError_t init_tiled()
{
    cudaFuncAttributes attr;                 // (asking for them loads the kernel: a first call may be inside a capture)
    cudaError_t e = cudaFuncGetAttributes(&attr, group_kernel);
    if (e != cudaSuccess) return e;
    e = init_vec<true>();
    return e != cudaSuccess ? e : init_vec<false>();
}

cudaError_t launch_shrink(cudaStream_t st, const Groups& g, const Adapters& ad, bool down, bool scaled, const float* x,
                          float* out, int rows, int L, bool early, int num_sms)
{
    ShrinkParams p;
    p.g = g;
    p.x = x;
    p.w = down ? ad.a : ad.b;
    p.scale = scaled ? ad.scale : nullptr;
    p.out = out;
    p.rows = rows; p.L = L; p.rank = ad.rank;
    const bool vec = L % 4 == 0 && aligned16(x) && aligned16(p.w) && (down || ad.rank % 4 == 0);
    const int tiles = g.perm ? g.max_tiles : (rows + TM - 1) / TM;
    if (down) {
        if (ad.rank <= 8)  return launch_shrink_t<8, true>(st, p, tiles, vec, early, num_sms);
        if (ad.rank <= 16) return launch_shrink_t<16, true>(st, p, tiles, vec, early, num_sms);
        if (ad.rank <= 32) return launch_shrink_t<32, true>(st, p, tiles, vec, early, num_sms);
        return launch_shrink_t<64, true>(st, p, tiles, vec, early, num_sms);
    }
    if (ad.rank <= 8)  return launch_shrink_t<8, false>(st, p, tiles, vec, early, num_sms);
    if (ad.rank <= 16) return launch_shrink_t<16, false>(st, p, tiles, vec, early, num_sms);
    if (ad.rank <= 32) return launch_shrink_t<32, false>(st, p, tiles, vec, early, num_sms);
    return launch_shrink_t<64, false>(st, p, tiles, vec, early, num_sms);
}

cudaError_t launch_expand(cudaStream_t st, const Groups& g, const Adapters& ad, bool up, bool scaled, const float* t,
                          float* c, int rows, int J, int act, bool early, bool wait_first, int num_sms)
{
    ExpandParams p;
    p.g = g;
    p.t = t;
    p.w = up ? ad.b : ad.a;
    p.scale = scaled ? ad.scale : nullptr;
    p.c = c;
    p.rows = rows; p.J = J; p.rank = ad.rank; p.act = act; p.wait_first = wait_first;
    const bool vec = J % 4 == 0 && aligned16(c) && (up || aligned16(p.w));
    const int tiles = g.perm ? g.max_tiles : (rows + TM - 1) / TM, cols = (J + EN - 1) / EN;
    // column tiles per CTA: as many as leave six CTAs per SM
    const long long per = static_cast<long long>(tiles) * cols / (6ll * num_sms);
    p.tiles_per = static_cast<int>(per < 1 ? 1 : per > 8 ? 8 : per);
    const dim3 grid(tiles, (cols + p.tiles_per - 1) / p.tiles_per, 1);
    if (up) {
        if (ad.rank <= 8)  return launch_expand_t<8, true>(st, p, grid, vec, early);
        if (ad.rank <= 16) return launch_expand_t<16, true>(st, p, grid, vec, early);
        return launch_expand_t<32, true>(st, p, grid, vec, early);
    }
    if (ad.rank <= 8)  return launch_expand_t<8, false>(st, p, grid, vec, early);
    if (ad.rank <= 16) return launch_expand_t<16, false>(st, p, grid, vec, early);
    return launch_expand_t<32, false>(st, p, grid, vec, early);
}

cudaError_t launch_outer(cudaStream_t st, const Groups& g, const Adapters& ad, const float* dt, const float* x, float* da,
                         const float* grad, const float* t, float* db, int rows, int N, int K, bool t_is_new,
                         bool early, int num_sms)
{
    OuterParams p;
    p.g = g;
    p.rows = rows;
    p.rank = ad.rank;
    int jobs = 0;
    p.job[0].tiles = p.job[1].tiles = 0;
    bool vec = ad.rank % 4 == 0;
    if (da) {
        p.job[jobs++] = OuterJob{dt, x, da, nullptr, K, 0, (K + 127) / 128, t_is_new ? 0 : 1};
        vec = vec && K % 4 == 0 && aligned16(x) && aligned16(dt);
    }
    if (db) {
        p.job[jobs++] = OuterJob{t, grad, db, ad.scale, N, 1, (N + 127) / 128, t_is_new || !da ? 1 : 0};
        vec = vec && N % 4 == 0 && aligned16(grad) && aligned16(t);
    }
    if (jobs == 0) return cudaSuccess;
    if (jobs == 1) { p.job[1] = p.job[0]; p.job[1].tiles = 0; }
    const int groups = g.perm ? ad.count : 1;
    if (ad.rank <= 8)  return launch_outer_t<8>(st, p, groups, ad.count, vec, early, num_sms);
    if (ad.rank <= 16) return launch_outer_t<16>(st, p, groups, ad.count, vec, early, num_sms);
    if (ad.rank <= 32) return launch_outer_t<32>(st, p, groups, ad.count, vec, early, num_sms);
    return launch_outer_t<64>(st, p, groups, ad.count, vec, early, num_sms);
}

}  // namespace lora
}  // namespace tt
