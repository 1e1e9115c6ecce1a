// Host entries of the low-rank adapter kernels (lora.cu), called by tt_lora_fwd / tt_lora_bwd.
#pragma once
#include <cuda_runtime.h>

namespace tt {
namespace lora {

constexpr int MAX_RANK = 128, MAX_ADAPTERS = 4096;
constexpr int TM = 64;                    // rows of one row tile (all of one adapter)

// The adapters of a call.
struct Adapters {
    const float* a;       // (count, rank, K)
    const float* b;       // (count, N, rank)
    const float* scale;   // (count) or null: 1
    int count, rank;
};

// Rows grouped by adapter, in device memory: perm lists the rows adapter by adapter (ascending row index within
// one) and behind them the rows without one; offset[e] .. offset[e + 1] is adapter e's range of it, entries `count` and
// `count` + 1 hold the range of the rows without an adapter.  perm null: every row has adapter 0, in its own order.
struct Groups {
    int* perm = nullptr;
    int* offset = nullptr;        // count + 2 entries
    int count = 0;                // adapters
    int max_tiles = 0;            // launch bound: at least the number of tiles
};

// Bytes of device memory the grouping of `rows` rows over `adapters` adapters takes, and its layout inside `mem`.
size_t groups_bytes(int rows, int adapters);
Groups groups_layout(void* mem, int rows, int adapters);

// Groups the rows.  An index outside [-1, adapters) counts as -1 and records DEV_BAD_ADAPTER in *status.
cudaError_t launch_group(cudaStream_t st, const Groups& g, const int* row_adapter, int rows, int adapters,
                         unsigned int* status);

// `early`: the launch directly in front, on the same stream, is one of this file's and of the same call; the two then
// overlap.  `wait_first`: it is the one that writes t or c.  `t_is_new`: it is the one that writes t (else dt, if any).

// out[m, r] = (scaled ? scale[e_m] : 1) * sum_l x[m, l] * W_e[r, l], zeros for rows without an adapter.  W = ad.a
// (down = true, L = K) or the transposed view of ad.b (down = false, L = N).
cudaError_t launch_shrink(cudaStream_t st, const Groups& g, const Adapters& ad, bool down, bool scaled, const float* x,
                          float* out, int rows, int L, bool early, int num_sms);

// c[m, j] = act(c[m, j] + (scaled ? scale[e_m] : 1) * sum_r t[m, r] * W_e[j, r]), W = ad.b (up = true, J = N) or the
// transposed view of ad.a (up = false, J = K).
cudaError_t launch_expand(cudaStream_t st, const Groups& g, const Adapters& ad, bool up, bool scaled, const float* t,
                          float* c, int rows, int J, int act, bool early, bool wait_first, int num_sms);

// da[e] = sum over e's rows of dt[m]^T x[m]   (rank, K)      skipped when da is null
// db[e] = scale[e] * sum over e's rows of g[m]^T t[m]  (N, rank)      skipped when db is null
cudaError_t launch_outer(cudaStream_t st, const Groups& g, const Adapters& ad, const float* dt, const float* x, float* da,
                         const float* grad, const float* t, float* db, int rows, int N, int K, bool t_is_new,
                         bool early, int num_sms);

// The forward pass of at most MAX_FEW_ROWS rows in two launches (lora_rows.cu), without a grouping; *taken = false, and
// nothing enqueued, when the call is outside what they hold.  t: (M, rank), always written.
constexpr int MAX_FEW_ROWS = 64;
constexpr int MAX_ROWS_SMEM = 224 * 1024;
cudaError_t launch_rows(cudaStream_t st, const Adapters& ad, const int* row_adapter, const float* x, const float* w,
                        const float* bias, float* y, float* t, int M, int N, int K, int act, unsigned int* status, int num_sms,
                        bool* taken);
// The backward pass of a small layer's adapters in one launch (lora_small.cu): dx, da and db may each be null, t is given
// when db is.  small_fits: whether the shape is one it holds.
bool small_fits(int M, int N, int K, int rank, int count);
cudaError_t launch_bwd_small(cudaStream_t st, const Adapters& ad, const int* row_adapter, const float* x, const float* w,
                             const float* y, const float* dy, const float* t, float* dx, float* da, float* db, int M, int N, int K,
                             int act, unsigned int* status);

// Kernel attributes, once per context (called from tt_create).
cudaError_t init_small();
cudaError_t init_tiled();
cudaError_t init_rows();

}  // namespace lora
}  // namespace tt
