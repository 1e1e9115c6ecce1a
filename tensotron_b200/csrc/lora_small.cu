// Backward of a small layer's low-rank adapters as ONE launch, the counterpart of linear_small.cuh.
//
// For the layers of small networks the tiled form's launches are each a few microseconds around well under a microsecond of
// arithmetic.  Here one grid computes all outputs, each CTA one of three kinds of tile, 32 columns wide:
//     dx  32 rows          dx = (dx or g w) + dt A        with dt = s g B formed for its own rows
//     dA  one adapter      dA = sum over its rows of dt x^T, dt formed for all its rows
//     dB  one adapter      dB = s sum over its rows of g t^T
// g = dy act'(y) is formed in shared memory and dt is formed again by every CTA that needs it, so nothing passes between CTAs.  Sums
// run in ascending index order; the eight row parts of dA and dB are added in order.
// 64 rows, 128 -> 64, rank 4, ReLU: 14.4 us per call against 20.6 us in five launches; 64 -> 64, rank 8, four adapters: 12.4
// against 26.7; 256 -> 128, rank 16: 21.5 against 34.3.  Everything a CTA reads is asked for at once and waited for once (with
// the operands read from global memory inside unrolled loops: 16.5 us for the first).
#include "lora.h"

#include <stdint.h>

#include "elementwise.cuh"
#include "lora_common.cuh"

namespace tt {
namespace lora {
namespace {

constexpr int THREADS = 256, TC = 32, PARTS = THREADS / TC, ROWS = 32;
constexpr int MAX_R = 16, MAX_M = 256, MAX_N = 256;                     // rank, rows, outputs
constexpr int MAX_G = 8192, MAX_T = 4096, MAX_B = 8192, MAX_AR = 128;   // rows x N, rows x rank, adapters x N x rank, adapters x rank
constexpr int MAX_COUNT = 16;
constexpr long long MAX_WORK = 1ll << 21;                               // rows x N x K, as for a Linear's backward in one launch
constexpr int SMEM_BYTES = (MAX_G + MAX_T + MAX_N * TC + MAX_B + MAX_AR * TC + PARTS * MAX_R * TC + MAX_M) * 4;

struct SmallParams {
    const float* a;
    const float* b;
    const float* scale;
    const int* row_adapter;
    const float* x;
    const float* w;
    const float* y;
    const float* dy;
    const float* t;
    float* dx;
    float* da;
    float* db;
    unsigned int* status;
    int M, N, K, rank, count, act;
    int tiles_dx, tiles_k, tiles_n, tiles_da;    // CTAs of dx, 32-column tiles of K and N, CTAs of dA
};

// Copies `rows` rows of up to TC columns (the first `n` of them exist) to shared memory, TC apart.
__device__ __forceinline__ void copy_columns(float* dst, const float* src, int rows, long long pitch, int n)
{
    const int c = threadIdx.x % TC;
    if (c < n)
#pragma unroll 2
        for (int r = threadIdx.x / TC; r < rows; r += PARTS) copy1(dst + r * TC + c, src + r * pitch + c, true);
}

__global__ void __launch_bounds__(THREADS) bwd_small_kernel(const SmallParams p)
{
    extern __shared__ __align__(128) float smem[];
    float* gs = smem;                       // g: the rows at hand x N (dB: x the tile's columns)
    float* ts = gs + MAX_G;                 // dt or t: the rows at hand x rank
    float* big = ts + MAX_T;                // 32 columns of w (dx) or x (dA)
    float* bs = big + MAX_N * TC;           // B of all adapters (dx) or of one (dA): [N][rank]
    float* as_ = bs + MAX_B;                // 32 columns of A of all adapters (dx)
    float* red = as_ + MAX_AR * TC;         // [part][rank][column]
    int* es = reinterpret_cast<int*>(red + PARTS * MAX_R * TC);
    const int tid = threadIdx.x, c = tid % TC, part = tid / TC;
    int tile = blockIdx.x;
    const int kind = tile < p.tiles_dx ? 0 : tile < p.tiles_dx + p.tiles_da ? 1 : 2;
    tile -= kind == 0 ? 0 : kind == 1 ? p.tiles_dx : p.tiles_dx + p.tiles_da;
    const int cols = kind == 2 ? p.tiles_n : p.tiles_k;
    const int c0 = (tile % cols) * TC, e = tile / cols;              // e: the adapter (dx: the row block)
    const int m0 = kind == 0 ? e * ROWS : 0, rows = kind == 0 ? min(ROWS, p.M - m0) : p.M;
    const int width = (kind == 2 ? p.N : p.K) - c0;                  // columns of this tile that exist, and perhaps more

    // everything is asked for at once: the kernel is a chain of latencies, and this is the only one through memory
    if (kind == 0) {
        if (p.w) copy_columns(big, p.w + c0, p.N, p.K, width);
        copy_columns(as_, p.a + c0, p.count * p.rank, p.K, width);
        for (int i = tid; i < p.count * p.N * p.rank; i += THREADS) copy1(bs + i, p.b + i, true);
    } else if (kind == 1) {
        copy_columns(big, p.x + c0, rows, p.K, width);
        for (int i = tid; i < p.N * p.rank; i += THREADS) copy1(bs + i, p.b + e * p.N * p.rank + i, true);
    } else {
        for (int i = tid; i < rows * p.rank; i += THREADS) copy1(ts + i, p.t + i, true);
    }
    bool bad = false;
    for (int m = tid; m < rows; m += THREADS) {
        const int k = p.row_adapter ? __ldg(p.row_adapter + m0 + m) : 0;
        const bool has = k >= 0 && k < p.count;
        bad |= !has && k != -1;
        es[m] = has ? k : -1;
    }
    if (bad && p.status) atomicCAS(p.status, 0u, static_cast<unsigned int>(DEV_BAD_ADAPTER));
    const int gw = kind == 2 ? min(TC, p.N) : p.N, g0 = kind == 2 ? c0 : 0;    // columns of g in shared memory (rows x gw <= MAX_G)
#pragma unroll 4
    for (int i = tid; i < rows * gw; i += THREADS) {
        const int m = i / gw, n = g0 + i - m * gw;
        const int at = (m0 + m) * p.N + n;
        gs[i] = n < p.N ? ew::act_grad(p.act ? __ldg(p.y + at) : 0.f, __ldg(p.dy + at), p.act) : 0.f;
    }
    commit_copies();
    wait_copies<0>();
    __syncthreads();

    if (kind != 2) {
        // dt of the rows at hand (dA: of its adapter's)
        for (int i = tid; i < rows * p.rank; i += THREADS) {
            const int m = i / p.rank, r = i - m * p.rank, k = es[m];
            float s = 0.f;
            if (k >= 0 && (kind == 0 || k == e)) {
                const float* b = bs + (kind == 0 ? k * p.N * p.rank : 0) + r;
                const float* g = gs + m * p.N;
#pragma unroll 4
                for (int n = 0; n < p.N; n++) s = fmaf(g[n], b[n * p.rank], s);
                if (p.scale) s *= __ldg(p.scale + k);
            }
            ts[i] = s;
        }
    }
    const int col = c0 + c;
    if (kind == 0) {
        constexpr int PER = ROWS / PARTS;               // rows part, part + PARTS, ... (those behind the last read the last)
        float acc[PER] = {};
        if (p.w && c < width) {
            const float* g[PER];
#pragma unroll
            for (int i = 0; i < PER; i++) g[i] = gs + min(part + i * PARTS, rows - 1) * p.N;
#pragma unroll 4
            for (int n = 0; n < p.N; n++) {
                const float wv = big[n * TC + c];
#pragma unroll
                for (int i = 0; i < PER; i++) acc[i] = fmaf(g[i][n], wv, acc[i]);
            }
        }
        __syncthreads();
        if (c >= width) return;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int m = part + i * PARTS;
            if (m >= rows) break;
            float* out = p.dx + (m0 + m) * p.K + col;
            float low = 0.f;
            if (es[m] >= 0)
                for (int r = 0; r < p.rank; r++) low = fmaf(ts[m * p.rank + r], as_[(es[m] * p.rank + r) * TC + c], low);
            *out = (p.w ? acc[i] : *out) + low;
        }
        return;
    }
    __syncthreads();
    float acc[MAX_R] = {};
    for (int m = part; m < rows; m += PARTS) {
        if (es[m] != e || c >= width) continue;
        const float v = kind == 2 ? gs[m * gw + c] : big[m * TC + c];
#pragma unroll
        for (int r = 0; r < MAX_R; r++)
            if (r < p.rank) acc[r] = fmaf(ts[m * p.rank + r], v, acc[r]);
    }
#pragma unroll
    for (int r = 0; r < MAX_R; r++)
        if (r < p.rank) red[(part * MAX_R + r) * TC + c] = acc[r];
    __syncthreads();
    const float scale = kind == 2 && p.scale ? __ldg(p.scale + e) : 1.f;
    for (int i = tid; i < p.rank * TC; i += THREADS) {
        // (neighbouring threads write neighbouring addresses: dA is (rank, K), dB (N, rank))
        const int r = kind == 2 ? i % p.rank : i / TC, cc = kind == 2 ? i / p.rank : i % TC;
        if (cc >= width) continue;
        float s = red[r * TC + cc];
#pragma unroll
        for (int q = 1; q < PARTS; q++) s += red[(q * MAX_R + r) * TC + cc];
        if (kind == 2) p.db[(e * p.N + c0 + cc) * p.rank + r] = scale * s;
        else           p.da[static_cast<long long>(e * p.rank + r) * p.K + c0 + cc] = s;
    }
}

}  // namespace

cudaError_t init_small() { return cudaFuncSetAttribute(bwd_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES); }

bool small_fits(int M, int N, int K, int rank, int count)
{
    return M <= MAX_M && N <= MAX_N && rank <= MAX_R && count <= MAX_COUNT && M * N <= MAX_G && M * rank <= MAX_T &&
           count * N * rank <= MAX_B && count * rank <= MAX_AR && static_cast<long long>(M) * N * K <= MAX_WORK;
}

cudaError_t launch_bwd_small(cudaStream_t st, const Adapters& ad, const int* row_adapter, const float* x, const float* w,
                             const float* y, const float* dy, const float* t, float* dx, float* da, float* db, int M, int N, int K,
                             int act, unsigned int* status)
{
    SmallParams p{ad.a, ad.b, ad.scale, row_adapter, x, w, y, dy, t, dx, da, db, status, M, N, K, ad.rank, ad.count, act, 0, 0, 0, 0};
    p.tiles_k = (K + TC - 1) / TC;
    p.tiles_n = (N + TC - 1) / TC;
    p.tiles_dx = dx ? (M + ROWS - 1) / ROWS * p.tiles_k : 0;
    p.tiles_da = da ? ad.count * p.tiles_k : 0;
    const int grid = p.tiles_dx + p.tiles_da + (db ? ad.count * p.tiles_n : 0);
    if (grid == 0) return cudaSuccess;
    bwd_small_kernel<<<grid, THREADS, SMEM_BYTES, st>>>(p);
    return cudaGetLastError();
}

}  // namespace lora
}  // namespace tt
