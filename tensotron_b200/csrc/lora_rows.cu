// Forward pass of a few rows (single tokens, decode batches) through a projection with low-rank adapters:
//     t[m] = A[e_m] x[m],    y[m] = act(w x[m] + bias + s[e_m] B[e_m] t[m])
// in two launches.  The projection is a stream of w (4 N K bytes, read once for 16 rows), the adapters a few megabytes
// beside it, so w's stream has to start at once and nothing may wait in front of it:
//     rows_down_kernel   t, one CTA per row and four ranks.  It lets the next launch begin right away.
//     rows_kernel        begins to stream w while t is still being formed, and waits for it only in front of its epilogue.
// A warp owns NR rows of w over the whole (or the CTA's share of the) contraction, its lanes four adjacent k each; x sits in
// shared memory in pairs of rows, where one 128-bit load feeds 4 NR multiply-adds (2 NR packed ones).  NR x MT sums per lane are added over the lanes by a
// transposing tree (NR x MT shuffles in all).  Where x does not fit, or where cutting N alone leaves SMs idle, the CTAs of
// a cluster cut k, and their sums are added through distributed shared memory in rank order.
// 4096 -> 4096, rank 16, per call: one row 24 us, 16 rows with an adapter each 28.7, 32 rows 47, 64 rows 86 (tiled form: 136, 146, 151,
// 155).  One row is bound by its 67 MB (10.3 us at the copy rate; a bare stream by the same copies takes 14.4) and about 4 us
// in front of and behind it, 64 rows by multiply-adds (28.9 us at the peak) and w coming from L2 four times.
#include "lora.h"

#include <cooperative_groups.h>
#include <stdint.h>

#include "lora_common.cuh"

namespace tt {
namespace lora {
namespace {

namespace cg = cooperative_groups;

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_X_BYTES = 128 * 1024;      // of shared memory for a CTA's share of x

struct RowsParams {
    const float* x;           // (M, K)
    const float* w;           // (N, K), or null: y holds the projection
    const float* bias;        // (N) or null
    const float* a;           // (count, rank, K)
    const float* b;           // (count, N, rank)
    const float* scale;       // (count) or null
    const int* row_adapter;   // (M) or null
    float* y;                 // (M, N)
    float* t;                 // (M, rank)
    unsigned int* status;
    int M, N, K, rank, count, act;
    int passes, kspan;        // row groups per warp; k per CTA of a cluster (a multiple of 128)
    int stages;               // steps of 128 k of the ring of w, 2 .. MAX_STAGES
};

__device__ __forceinline__ int adapter_of(const RowsParams& p, int m)
{
    return p.row_adapter ? __ldg(p.row_adapter + m) : 0;
}

template <bool VEC>
__device__ __forceinline__ float4 ld4(const float* p, int n)
{
    if (n <= 0) return make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC) return __ldg(reinterpret_cast<const float4*>(p));
    return make_float4(__ldg(p), n > 1 ? __ldg(p + 1) : 0.f, n > 2 ? __ldg(p + 2) : 0.f, n > 3 ? __ldg(p + 3) : 0.f);
}

// Waits until at most `n` of the calling thread's copy groups are unfinished.
__device__ __forceinline__ void wait_copies_n(int n)
{
    switch (n) {
    case 0: wait_copies<0>(); break;
    case 1: wait_copies<1>(); break;
    case 2: wait_copies<2>(); break;
    case 3: wait_copies<3>(); break;
    default: wait_copies<4>(); break;
    }
}

constexpr int MAX_CLUSTER = 8;
constexpr int MAX_STAGES = 6;        // of the ring of w (wait_copies_n knows up to MAX_STAGES - 2)

constexpr int DOWN_RANKS = 4;

template <bool VEC>
__global__ void __launch_bounds__(THREADS) rows_down_kernel(const RowsParams p)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ float red[WARPS][DOWN_RANKS];
    const int m = blockIdx.y, r0 = blockIdx.x * DOWN_RANKS, tid = threadIdx.x;
    const int e = adapter_of(p, m);
    const bool has = e >= 0 && e < p.count;
    if (!has && e != -1 && tid == 0 && p.status) atomicCAS(p.status, 0u, static_cast<unsigned int>(DEV_BAD_ADAPTER));
    float acc[DOWN_RANKS] = {};
    if (has) {
        const float* x = p.x + static_cast<long long>(m) * p.K;
        const float* a = p.a + (static_cast<long long>(e) * p.rank + r0) * p.K;
#pragma unroll 4
        for (int k = tid * 4; k < p.K; k += THREADS * 4) {
            const float4 xv = ld4<VEC>(x + k, p.K - k);
#pragma unroll
            for (int j = 0; j < DOWN_RANKS; j++) {
                const float4 av = ld4<VEC>(a + static_cast<long long>(j) * p.K + k, r0 + j < p.rank ? p.K - k : 0);
                acc[j] = fmaf(xv.x, av.x, acc[j]);
                acc[j] = fmaf(xv.y, av.y, acc[j]);
                acc[j] = fmaf(xv.z, av.z, acc[j]);
                acc[j] = fmaf(xv.w, av.w, acc[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < DOWN_RANKS; j++) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
        if ((tid & 31) == 0) red[tid >> 5][j] = acc[j];
    }
    __syncthreads();
    if (tid < DOWN_RANKS && r0 + tid < p.rank) {
        float s = red[0][tid];
#pragma unroll
        for (int w = 1; w < WARPS; w++) s += red[w][tid];
        p.t[static_cast<long long>(m) * p.rank + r0 + tid] = s;
    }
}

template <int NR, int MT, bool VEC>
__global__ void __launch_bounds__(THREADS) rows_kernel(const RowsParams p)
{
    // Up to eight rows keep two sums per output, over the even and the odd k, so that a 128-bit piece of w and one of x
    // make two packed multiply-adds per output.  Sixteen rows would need 2 x 16 x NR registers for that: they go in pairs, x
    // is stored pair by pair, and a packed multiply-add serves two rows.
    constexpr bool PAIRS = MT > 8;
    constexpr int NA = PAIRS ? MT / 2 : MT, VALUES = WARPS * NR * MT;
    extern __shared__ __align__(128) float rows_smem[];
    __shared__ int adapter_s[MT];
    __shared__ float scale_s[MT];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int m0 = blockIdx.y * MT, mn = min(MT, p.M - m0);
    float* xs = rows_smem;                             // [MT][kspan], or pairs (see below)
    float* red = xs + (p.w ? MT * p.kspan : 0);        // [2][C][this CTA's share of the sums]
    float* ts = red + 2 * (VALUES + MAX_CLUSTER);      // [MT][rank]
    float* ring = ts + ((MT * p.rank + 3) & ~3);       // [stages][WARPS][NR][128]
    const int k0 = rank * p.kspan, k1 = min(p.K, k0 + p.kspan);
    const long long row0 = static_cast<long long>(blockIdx.x / C) * p.passes * WARPS * NR;
    const int steps = p.w && k1 > k0 ? (k1 - k0 + 127) / 128 : 0;
    const int total = steps * p.passes;
    const int share = (WARPS * NR * mn + C - 1) / C;   // of a pass's sums: what one CTA of the cluster finishes

    int e_own = -1;
    if (tid < mn) e_own = adapter_of(p, m0 + tid);
    // Every lane copies the four k of each of its warp's rows that it will read itself, `stages` - 1 steps ahead: no
    // barrier is needed for w, and the bytes in flight do not take registers.  Rows behind the last one are read as
    // the last one (their sums are not stored).
    // The warps begin at different steps and wrap around: rows of w are often a power of two apart, and warps that walk
    // them from the same offset in lockstep keep hitting the same memory channels.
    const int rot = steps > 0 ? static_cast<int>((blockIdx.x / C * WARPS + warp) % static_cast<unsigned int>(steps)) : 0;
    int is_step = rot, is_slot = 0, issued = 0, left_in_pass = steps;
    long long is_row = row0 + warp * NR;
    const float* src[NR];
    const auto rows_from = [&](long long n) {
#pragma unroll
        for (int i = 0; i < NR; i++) src[i] = p.w + min(n + i, static_cast<long long>(p.N) - 1) * p.K + k0 + lane * 4;
    };
    const auto issue = [&]() {
        if (issued < total) {
            const int at = is_step * 128, left = k1 - k0 - lane * 4 - at;
            float* dst = ring + ((is_slot * WARPS + warp) * NR) * 128 + lane * 4;
#pragma unroll
            for (int i = 0; i < NR; i++) copy4(dst + i * 128, left > 0 ? src[i] + at : p.w, left, VEC);
            issued++;
            if (++is_slot == p.stages) is_slot = 0;
            if (++is_step == steps) is_step = 0;
            if (--left_in_pass == 0) {
                left_in_pass = steps;
                is_row += WARPS * NR;
                rows_from(is_row);
            }
        }
        commit_copies();
    };
    if (steps > 0) {
        rows_from(is_row);
        const int q4 = p.kspan / 4;
        if constexpr (PAIRS) {
            // xs[pair][step][k 0,1 | k 2,3 of the lane][lane]: (row 0, row 1) of one k, then of the next.  Only the first step of
            // w is asked for in front of x: x behind a full ring would arrive last.
            issue();
#pragma unroll 4
            for (int i = tid; i < NA * q4; i += THREADS) {
                const int j = i / q4, q = i - j * q4, k = k0 + q * 4;
                const float* xr = p.x + static_cast<long long>(m0 + 2 * j) * p.K + k;
                const float4 u = ld4<VEC>(xr, 2 * j < mn ? k1 - k : 0);
                const float4 v = ld4<VEC>(xr + p.K, 2 * j + 1 < mn ? k1 - k : 0);
                float* dst = xs + (j * p.kspan + (q & ~31) * 4) * 2 + (q & 31) * 4;
                *reinterpret_cast<float4*>(dst) = make_float4(u.x, v.x, u.y, v.y);
                *reinterpret_cast<float4*>(dst + 128) = make_float4(u.z, v.z, u.w, v.w);
            }
            for (int s = 1; s + 1 < p.stages; s++) issue();
        } else {
            for (int i = tid; i < MT * q4; i += THREADS) {
                const int m = i / q4, k = k0 + (i - m * q4) * 4, left = m < mn ? k1 - k : 0;
                copy4(xs + i * 4, left > 0 ? p.x + static_cast<long long>(m0 + m) * p.K + k : p.x, left, VEC);
            }
            for (int s = 0; s + 1 < p.stages; s++) issue();       // (x arrives with the first step)
            wait_copies_n(p.stages - 2);
        }
    }
    if (tid < MT) adapter_s[tid] = e_own >= 0 && e_own < p.count ? e_own : -1;
    __syncthreads();
    if (tid < MT) scale_s[tid] = adapter_s[tid] < 0 ? 0.f : p.scale ? __ldg(p.scale + adapter_s[tid]) : 1.f;
    // what the first epilogue will read of B comes to L2 meanwhile
    for (int q = rank * share + tid; q < min((rank + 1) * share, WARPS * NR * mn); q += THREADS) {
        const int m = q / (WARPS * NR), e = adapter_s[m];
        const long long n = row0 + (q - m * (WARPS * NR));
        if (e >= 0 && n < p.N)
            for (int r = 0; r < p.rank; r += 32)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(p.b + (static_cast<long long>(e) * p.N + n) * p.rank + r));
    }
    int slot = 0;
    for (int pass = 0; pass < p.passes; pass++) {
        const long long n0 = row0 + pass * WARPS * NR;
        float2 acc2[NR][NA];
#pragma unroll
        for (int i = 0; i < NR; i++)
#pragma unroll
            for (int j = 0; j < NA; j++) acc2[i][j] = make_float2(0.f, 0.f);
        for (int done = 0, s = rot; done < steps; done++, s = s + 1 == steps ? 0 : s + 1) {
            __syncwarp();          // (lanes that ran ahead alone would ask for their pieces of w in requests of their own)
            wait_copies_n(p.stages - 2);
            const float* wp = ring + ((slot * WARPS + warp) * NR) * 128 + lane * 4;
            if (++slot == p.stages) slot = 0;
            float4 wv[NR];
#pragma unroll
            for (int i = 0; i < NR; i++) wv[i] = *reinterpret_cast<const float4*>(wp + i * 128);
            if constexpr (PAIRS) {
                const float* xp = xs + s * 256 + lane * 4;
#pragma unroll
                for (int j = 0; j < NA; j++) {
                    const float4 x01 = *reinterpret_cast<const float4*>(xp + j * 2 * p.kspan);
                    const float4 x23 = *reinterpret_cast<const float4*>(xp + j * 2 * p.kspan + 128);
#pragma unroll
                    for (int i = 0; i < NR; i++) acc2[i][j] = __ffma2_rn(make_float2(wv[i].x, wv[i].x), make_float2(x01.x, x01.y), acc2[i][j]);
#pragma unroll
                    for (int i = 0; i < NR; i++) acc2[i][j] = __ffma2_rn(make_float2(wv[i].y, wv[i].y), make_float2(x01.z, x01.w), acc2[i][j]);
#pragma unroll
                    for (int i = 0; i < NR; i++) acc2[i][j] = __ffma2_rn(make_float2(wv[i].z, wv[i].z), make_float2(x23.x, x23.y), acc2[i][j]);
#pragma unroll
                    for (int i = 0; i < NR; i++) acc2[i][j] = __ffma2_rn(make_float2(wv[i].w, wv[i].w), make_float2(x23.z, x23.w), acc2[i][j]);
                }
            } else {
                const float* xp = xs + s * 128 + lane * 4;
#pragma unroll
                for (int j = 0; j < NA; j++) {
                    const float4 xv = *reinterpret_cast<const float4*>(xp + j * p.kspan);
#pragma unroll
                    for (int i = 0; i < NR; i++) acc2[i][j] = __ffma2_rn(make_float2(wv[i].x, wv[i].y), make_float2(xv.x, xv.y), acc2[i][j]);
#pragma unroll
                    for (int i = 0; i < NR; i++) acc2[i][j] = __ffma2_rn(make_float2(wv[i].z, wv[i].w), make_float2(xv.z, xv.w), acc2[i][j]);
                }
            }
            issue();
        }
        float acc[NR][MT];
#pragma unroll
        for (int i = 0; i < NR; i++)
#pragma unroll
            for (int m = 0; m < MT; m++) {
                if constexpr (PAIRS) acc[i][m] = m & 1 ? acc2[i][m / 2].y : acc2[i][m / 2].x;
                else                 acc[i][m] = acc2[i][m].x + acc2[i][m].y;
            }
        // transposing tree: with each step a lane keeps half of the m it holds
        int o = 16, mine = 0;
#pragma unroll
        for (int h = MT / 2; h > 0; h >>= 1, o >>= 1) {
            const bool up = (lane & o) != 0;
            if (up) mine += h;
#pragma unroll
            for (int i = 0; i < NR; i++)
#pragma unroll
                for (int m = 0; m < h; m++) {
                    const float send = up ? acc[i][m] : acc[i][m + h];
                    const float keep = up ? acc[i][m + h] : acc[i][m];
                    acc[i][m] = keep + __shfl_xor_sync(0xffffffffu, send, o);
                }
        }
        for (; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < NR; i++) acc[i][0] += __shfl_xor_sync(0xffffffffu, acc[i][0], o);
        // Each sum goes to the CTA that finishes it (two buffers in turn: one barrier per pass is enough, and nobody reads
        // another CTA's memory after it).
        if (C > 1 && pass == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");    // all CTAs have started
        float* mine_red = red + (pass & 1) * (VALUES + MAX_CLUSTER);
        if ((lane & (32 / MT - 1)) == 0 && mine < mn) {
#pragma unroll
            for (int i = 0; i < NR; i++) {
                const int q = mine * (WARPS * NR) + warp * NR + i, owner = q / share;
                float* dst = mine_red + rank * share + (q - owner * share);
                *(C > 1 ? cluster.map_shared_rank(dst, owner) : dst) = acc[i][0];
            }
        }
        if (pass == 0) {
            asm volatile("griddepcontrol.wait;" ::: "memory");        // t is complete from here on
            for (int i = tid; i < mn * p.rank; i += THREADS) ts[i] = __ldcg(p.t + static_cast<long long>(m0) * p.rank + i);
        }
        if (C > 1) cluster.sync(); else __syncthreads();
        for (int q = rank * share + tid; q < min((rank + 1) * share, WARPS * NR * mn); q += THREADS) {
            const int m = q / (WARPS * NR), row = q - m * (WARPS * NR);
            const long long n = n0 + row;
            if (n >= p.N) continue;
            float* out = p.y + static_cast<long long>(m0 + m) * p.N + n;
            float v = 0.f, u = 0.f;
            if (!p.w) v = *out;
            else if (p.bias) v = __ldg(p.bias + n);
            const int e = adapter_s[m];
            if (e >= 0) {
                const float* b = p.b + (static_cast<long long>(e) * p.N + n) * p.rank;
                const float* tr = ts + m * p.rank;
                if (VEC && (p.rank & 3) == 0) {
#pragma unroll 4
                    for (int r = 0; r < p.rank; r += 4) {
                        const float4 bv = __ldg(reinterpret_cast<const float4*>(b + r));
                        u = fmaf(tr[r], bv.x, u);
                        u = fmaf(tr[r + 1], bv.y, u);
                        u = fmaf(tr[r + 2], bv.z, u);
                        u = fmaf(tr[r + 3], bv.w, u);
                    }
                } else {
                    for (int r = 0; r < p.rank; r++) u = fmaf(tr[r], __ldg(b + r), u);
                }
                u *= scale_s[m];
            }
            if (p.w) {
                float z = mine_red[q - rank * share];
                for (int c = 1; c < C; c++) z += mine_red[c * share + q - rank * share];
                v = z + v;
            }
            *out = act_apply(v + u, p.act);
        }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int NR, int MT, bool VEC>
cudaError_t launch_rows_t(cudaStream_t st, const RowsParams& p, dim3 grid, int cluster, int smem, bool init)
{
    if (init)
        return cudaFuncSetAttribute(rows_kernel<NR, MT, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_ROWS_SMEM);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned int>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, rows_kernel<NR, MT, VEC>, p);
}

template <int MT, bool VEC>
cudaError_t launch_rows_m(int nr, cudaStream_t st, const RowsParams& p, dim3 grid, int cluster, int smem, bool init)
{
    if constexpr (VEC) {
        switch (nr) {
        case 1: return launch_rows_t<1, MT, VEC>(st, p, grid, cluster, smem, init);
        case 2: return launch_rows_t<2, MT, VEC>(st, p, grid, cluster, smem, init);
        case 3: return launch_rows_t<3, MT, VEC>(st, p, grid, cluster, smem, init);
        case 5: return launch_rows_t<5, MT, VEC>(st, p, grid, cluster, smem, init);
        case 6: return launch_rows_t<6, MT, VEC>(st, p, grid, cluster, smem, init);
        case 7: return launch_rows_t<7, MT, VEC>(st, p, grid, cluster, smem, init);
        case 8: return launch_rows_t<8, MT, VEC>(st, p, grid, cluster, smem, init);
        }
    }
    return launch_rows_t<4, MT, VEC>(st, p, grid, cluster, smem, init);
}

template <bool VEC>
cudaError_t launch_rows_v(int mt, int nr, cudaStream_t st, const RowsParams& p, dim3 grid, int cluster, int smem, bool init)
{
    switch (mt) {
    case 4: return launch_rows_m<4, VEC>(nr, st, p, grid, cluster, smem, init);
    case 8: return launch_rows_m<8, VEC>(nr, st, p, grid, cluster, smem, init);
    }
    return launch_rows_m<16, VEC>(nr, st, p, grid, cluster, smem, init);
}

}  // namespace

cudaError_t init_rows()
{
    cudaFuncAttributes attr;                 // (loads the kernels that need no attribute, as for the others)
    cudaError_t loaded = cudaFuncGetAttributes(&attr, rows_down_kernel<true>);
    if (loaded == cudaSuccess) loaded = cudaFuncGetAttributes(&attr, rows_down_kernel<false>);
    if (loaded != cudaSuccess) return loaded;
    const RowsParams none = {};
    for (int mt = 4; mt <= 16; mt *= 2) {
        for (int nr = 1; nr <= 8; nr++) {
            const cudaError_t e = launch_rows_v<true>(mt, nr, nullptr, none, dim3(1), 1, 0, true);
            if (e != cudaSuccess) return e;
        }
        const cudaError_t e = launch_rows_v<false>(mt, 4, nullptr, none, dim3(1), 1, 0, true);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_rows(cudaStream_t st, const Adapters& ad, const int* row_adapter, const float* x, const float* w,
                        const float* bias, float* y, float* t, int M, int N, int K, int act, unsigned int* status, int num_sms,
                        bool* taken)
{
    *taken = false;
    if (M > MAX_FEW_ROWS) return cudaSuccess;
    const int mt = M > 8 ? 16 : M > 4 ? 8 : 4;
    const bool vec = K % 4 == 0 && aligned16(x) && aligned16(ad.a) && (ad.rank % 4 != 0 || aligned16(ad.b)) && (!w || aligned16(w));
    // Cluster size, rows of w per warp and passes that give the busiest SM the least of w to read; the smallest cluster
    // wins a tie.
    int C = 0, nr = 1, passes = 1, kspan = 128;
    long long best = 0;
    for (int c = 1; c <= (w ? MAX_CLUSTER : 1); c *= 2) {
        const int span = ((K + c - 1) / c + 127) / 128 * 128;
        if (w && static_cast<long long>(span) * mt * 4 > MAX_X_BYTES) continue;
        if (c > 1 && span * (c - 1) >= K) break;                      // an empty share
        const long long warps = static_cast<long long>(num_sms / c) * WARPS;
        const int per = static_cast<int>((N + warps - 1) / warps);    // rows of w per warp
        const int ps = vec ? (per + 7) / 8 : (per + 3) / 4;
        const int r = vec ? (per + ps - 1) / ps : 4;
        const long long cost = static_cast<long long>(ps) * r * span;
        if (C == 0 || cost < best) { C = c; nr = r; passes = ps; kspan = span; best = cost; }
    }
    if (C == 0) return cudaSuccess;
    const int fixed = static_cast<int>(sizeof(float)) * ((w ? mt * kspan : 0) + 2 * (WARPS * nr * mt + MAX_CLUSTER) + ((mt * ad.rank + 3) & ~3));
    const int stage = static_cast<int>(sizeof(float)) * WARPS * nr * 128;
    int stages = w ? (MAX_ROWS_SMEM - fixed) / stage : 0;
    if (stages > MAX_STAGES) stages = MAX_STAGES;
    if (w && stages < 2) return cudaSuccess;
    RowsParams p{x, w, bias, ad.a, ad.b, ad.scale, row_adapter, y, t, status, M, N, K, ad.rank, ad.count, act, passes, kspan, stages};
    const dim3 down((ad.rank + DOWN_RANKS - 1) / DOWN_RANKS, M, 1);
    if (vec) rows_down_kernel<true><<<down, THREADS, 0, st>>>(p);
    else     rows_down_kernel<false><<<down, THREADS, 0, st>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int smem = fixed + stages * stage;
    const int per_cluster = passes * WARPS * nr;
    const dim3 grid(static_cast<unsigned int>((N + per_cluster - 1) / per_cluster) * C, (M + mt - 1) / mt, 1);
    *taken = true;
    return vec ? launch_rows_v<true>(mt, nr, st, p, grid, C, smem, false) : launch_rows_v<false>(mt, nr, st, p, grid, C, smem, false);
}

}  // namespace lora
}  // namespace tt
