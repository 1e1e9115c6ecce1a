// ClipGradNorm and Adam over lists of tensors.
//
// The lists travel as kernel parameters (pointer, size and first chunk of each tensor), so a call copies nothing to
// the device, keeps nothing and can be captured; a list longer than one table holds takes several launches.  A tensor
// is cut into chunks of CHUNK elements; the CTAs of a launch share out the chunks of all tensors evenly, so a list of a
// thousand small tensors costs what one tensor of their total size costs.
#include "tensor_lists.h"

#include <stdint.h>

#include "elementwise.cuh"

namespace tt {
namespace lists {
namespace {

constexpr int THREADS = 256;
constexpr int CHUNK = 4096;                 // elements per chunk: four 128-bit loads per thread

// Elements in front of the first 16-byte boundary (a tensor is at least 4-byte aligned).
__host__ __device__ inline int head_of(const void* p) { return static_cast<int>((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / 4; }

template <int CAP>
struct NormTable {
    int count, chunks;
    int first[CAP + 1];                     // first chunk of each tensor
    float* ptr[CAP];
    long long size[CAP];
};

template <int CAP>
struct AdamTable {
    int count, chunks;
    int first[CAP + 1];
    float* p[CAP];
    const float* g[CAP];
    float* m[CAP];
    float* v[CAP];
    long long size[CAP];
};

// The tensor that chunk `c` belongs to: the last one whose first chunk is at most c.
template <typename T>
__device__ __forceinline__ int tensor_of(const T& t, int c)
{
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= c) lo = mid; else hi = mid;
    }
    return lo;
}

// Calls body4(i) for every aligned group of four elements of chunk `c` of a tensor of `size` elements whose first
// `head` elements lie in front of the 16-byte boundary, and body1(i) for the elements outside such groups.
template <typename F4, typename F1>
__device__ __forceinline__ void for_chunk(int c, long long size, int head, F4 body4, F1 body1)
{
    const long long lo = head + static_cast<long long>(c) * CHUNK;
    const long long hi = lo + CHUNK < size ? lo + CHUNK : size;
    if (c == 0 && threadIdx.x < head && threadIdx.x < size) body1(static_cast<long long>(threadIdx.x));
    const long long n4 = hi > lo ? (hi - lo) >> 2 : 0;
    for (int q = threadIdx.x; q < n4; q += THREADS) body4(lo + 4ll * q);
    const long long t = lo + 4 * n4 + threadIdx.x;
    if (threadIdx.x < 4 && t < hi) body1(t);
}

__device__ __forceinline__ double square(float v) { return static_cast<double>(v) * static_cast<double>(v); }

// Sum of one value per thread: xor-shuffle tree, then the warps in order.
__device__ __forceinline__ double block_sum(double s, double* red)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < THREADS / 32; w++) t += red[w];
    __syncthreads();
    return t;
}

__device__ __forceinline__ float clip_coef(float norm, float max_norm, float eps)
{
    const float c = max_norm / (norm + eps);
    return c < 0.f ? 0.f : c > 1.f ? 1.f : c;       // a NaN stays one
}

struct NormFinish {
    double* partial;        // partial sums of all launches of the call
    int base, total;        // this launch's first one, and their number over the call
    int last_launch;
    unsigned int* ticket;
    float* norm_out;
    float* coef_out;        // (workspace word or the caller's)
    float max_norm, eps;
};

// partial[base + block] = sum of squares of this block's chunks, in double precision: a float gradient's square
// neither overflows nor vanishes, and the order of the sum hardly shows.  The last block to finish adds all partial
// sums in a fixed order.
template <int CAP>
__global__ void __launch_bounds__(THREADS) norm_kernel(const __grid_constant__ NormTable<CAP> t, const NormFinish f)
{
    __shared__ double red[THREADS / 32];
    __shared__ unsigned int last;
    double s = 0.0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const float* g = t.ptr[i];
        for_chunk(c - t.first[i], t.size[i], head_of(g),
                  [&](long long e) {
                      const float4 v = *reinterpret_cast<const float4*>(g + e);
                      s += (square(v.x) + square(v.y)) + (square(v.z) + square(v.w));
                  },
                  [&](long long e) { s += square(g[e]); });
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) {
        f.partial[f.base + blockIdx.x] = s;
        __threadfence();
        last = f.last_launch && atomicAdd(f.ticket, 1u) == gridDim.x - 1 ? 1u : 0u;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    s = 0.0;
    for (int i = threadIdx.x; i < f.total; i += THREADS) s += __ldcg(f.partial + i);
    s = block_sum(s, red);
    if (threadIdx.x == 0) {
        const float norm = static_cast<float>(sqrt(s));
        if (f.norm_out) *f.norm_out = norm;
        if (f.coef_out) *f.coef_out = clip_coef(norm, f.max_norm, f.eps);
        *f.ticket = 0u;
    }
}

template <int CAP>
__global__ void __launch_bounds__(THREADS) scale_kernel(const __grid_constant__ NormTable<CAP> t, const float* coef_ptr)
{
    const float coef = *coef_ptr;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = tensor_of(t, c);
        float* g = t.ptr[i];
        for_chunk(c - t.first[i], t.size[i], head_of(g),
                  [&](long long e) {
                      float4 v = *reinterpret_cast<const float4*>(g + e);
                      v.x *= coef; v.y *= coef; v.z *= coef; v.w *= coef;
                      *reinterpret_cast<float4*>(g + e) = v;
                  },
                  [&](long long e) { g[e] *= coef; });
    }
}

struct AdamArgs {
    float* adv;
    const float* grad_scale;
    float b1, b2, lr, eps, cwd, dfac;
    int advance, last_launch;
    unsigned int* ticket;
};

// Each CTA forms the bias corrections of this step itself; the last one to finish writes them to adv (every CTA has
// read the step counter by then).
template <int CAP>
__global__ void __launch_bounds__(THREADS) adam_kernel(const __grid_constant__ AdamTable<CAP> t, const AdamArgs a)
{
    __shared__ float fix[3];
    if (threadIdx.x == 0) {
        if (a.advance) {
            const float step = *a.adv + 1.f;
            fix[0] = step;
            fix[1] = 1.f / (1.f - powf(a.b1, step));
            fix[2] = 1.f / (1.f - powf(a.b2, step));
        } else {
            fix[1] = a.adv[1];
            fix[2] = a.adv[2];
        }
    }
    __syncthreads();
    const float ibc1 = fix[1], ibc2 = fix[2], omb1 = 1.f - a.b1, omb2 = 1.f - a.b2;
    const float coef = a.grad_scale ? *a.grad_scale : 1.f;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = tensor_of(t, c);
        float* p = t.p[i];
        const float* g = t.g[i];
        float* m = t.m[i];
        float* v = t.v[i];
        const int head = head_of(p);
        const bool vec = head_of(g) == head && head_of(m) == head && head_of(v) == head;
        const auto one = [&](long long e) {
            float pp = p[e], mm = m[e], vv = v[e];
            ew::adam_one(pp, coef * g[e], mm, vv, a.b1, omb1, a.b2, omb2, a.lr, a.eps, ibc1, ibc2, a.cwd, a.dfac);
            p[e] = pp; m[e] = mm; v[e] = vv;
        };
        for_chunk(c - t.first[i], t.size[i], vec ? head : 0,
                  [&](long long e) {
                      if (!vec) {
                          for (int k = 0; k < 4; k++) one(e + k);
                          return;
                      }
                      float4 pp = *reinterpret_cast<const float4*>(p + e);
                      float4 gg = *reinterpret_cast<const float4*>(g + e);
                      float4 mm = *reinterpret_cast<const float4*>(m + e);
                      float4 vv = *reinterpret_cast<const float4*>(v + e);
                      gg.x *= coef; gg.y *= coef; gg.z *= coef; gg.w *= coef;
                      ew::adam_one(pp.x, gg.x, mm.x, vv.x, a.b1, omb1, a.b2, omb2, a.lr, a.eps, ibc1, ibc2, a.cwd, a.dfac);
                      ew::adam_one(pp.y, gg.y, mm.y, vv.y, a.b1, omb1, a.b2, omb2, a.lr, a.eps, ibc1, ibc2, a.cwd, a.dfac);
                      ew::adam_one(pp.z, gg.z, mm.z, vv.z, a.b1, omb1, a.b2, omb2, a.lr, a.eps, ibc1, ibc2, a.cwd, a.dfac);
                      ew::adam_one(pp.w, gg.w, mm.w, vv.w, a.b1, omb1, a.b2, omb2, a.lr, a.eps, ibc1, ibc2, a.cwd, a.dfac);
                      *reinterpret_cast<float4*>(p + e) = pp;
                      *reinterpret_cast<float4*>(m + e) = mm;
                      *reinterpret_cast<float4*>(v + e) = vv;
                  },
                  one);
    }
    if (!a.last_launch || !a.advance) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        if (atomicAdd(a.ticket, 1u) == gridDim.x - 1) {
            a.adv[0] = fix[0];
            a.adv[1] = ibc1;
            a.adv[2] = ibc2;
            *a.ticket = 0u;
        }
    }
}

long long chunks_of(long long size, int head)
{
    const long long body = size - head;
    return size <= 0 ? 0 : body <= 0 ? 1 : (body + CHUNK - 1) / CHUNK;
}

// Grid of a launch over `chunks` chunks: at most eight CTAs per SM.
int grid_of(long long chunks, int num_sms)
{
    const long long cap = 8ll * num_sms;
    return static_cast<int>(chunks < 1 ? 1 : chunks < cap ? chunks : cap);
}

constexpr long long MAX_CHUNKS = 1ll << 30;          // of one launch: chunk numbers are ints

// Fills `t` with tensors from *at on; false when nothing is left.
template <int CAP>
bool fill(NormTable<CAP>& t, int count, float* const* ptr, const long long* sizes, int* at)
{
    t.count = t.chunks = 0;
    for (; *at < count && t.count < CAP; (*at)++) {
        const long long n = chunks_of(sizes[*at], head_of(ptr[*at]));
        if (n == 0) continue;
        if (t.count && t.chunks + n > MAX_CHUNKS) break;
        t.first[t.count] = t.chunks;
        t.ptr[t.count] = ptr[*at];
        t.size[t.count] = sizes[*at];
        t.count++;
        t.chunks += static_cast<int>(n);
    }
    t.first[t.count] = t.chunks;
    return t.count > 0;
}

template <int CAP>
cudaError_t clip_cap(cudaStream_t st, int count, float* const* grads, const long long* sizes, float max_norm, float eps,
                     bool scale, float* norm_out, float* coef_out, void* workspace, unsigned int* ticket, int num_sms,
                     long long* launches)
{
    double* partial = static_cast<double*>(workspace);
    float* coef = coef_out ? coef_out : reinterpret_cast<float*>(partial + MAX_PARTIALS);
    NormTable<CAP> t;
    int at = 0, base = 0;
    bool more = fill(t, count, grads, sizes, &at);
    do {
        int ahead = at;
        while (ahead < count && sizes[ahead] <= 0) ahead++;
        const bool last = !more || ahead >= count;
        // (a list of many tables shares the partial sums out among its launches)
        int grid = grid_of(t.chunks, num_sms);
        const int share = (MAX_PARTIALS - base) / ((count - at) / CAP + 2);
        if (grid > share) grid = share > 1 ? share : 1;
        const NormFinish f{partial, base, base + grid, last ? 1 : 0, ticket, norm_out, coef, max_norm, eps};
        norm_kernel<CAP><<<grid, THREADS, 0, st>>>(t, f);
        (*launches)++;
        base += grid;
        more = !last && fill(t, count, grads, sizes, &at);
    } while (more);
    if (scale) {
        at = 0;
        while (fill(t, count, grads, sizes, &at)) {
            scale_kernel<CAP><<<grid_of(t.chunks, num_sms), THREADS, 0, st>>>(t, coef);
            (*launches)++;
        }
    }
    return cudaGetLastError();
}

template <int CAP>
cudaError_t adam_cap(cudaStream_t st, int count, float* const* p, const float* const* g, float* const* m,
                     float* const* v, const long long* sizes, const AdamArgs& args, int num_sms, long long* launches)
{
    AdamTable<CAP> t;
    AdamArgs a = args;
    int at = 0;
    do {
        t.count = t.chunks = 0;
        for (; at < count && t.count < CAP; at++) {
            const int head = head_of(p[at]);
            const bool vec = head_of(g[at]) == head && head_of(m[at]) == head && head_of(v[at]) == head;
            const long long n = chunks_of(sizes[at], vec ? head : 0);
            if (n == 0) continue;
            if (t.count && t.chunks + n > MAX_CHUNKS) break;
            const int k = t.count++;
            t.first[k] = t.chunks;
            t.p[k] = p[at]; t.g[k] = g[at]; t.m[k] = m[at]; t.v[k] = v[at];
            t.size[k] = sizes[at];
            t.chunks += static_cast<int>(n);
        }
        t.first[t.count] = t.chunks;
        int ahead = at;
        while (ahead < count && sizes[ahead] <= 0) ahead++;
        at = ahead;
        a.last_launch = at >= count ? 1 : 0;
        adam_kernel<CAP><<<grid_of(t.chunks, num_sms), THREADS, 0, st>>>(t, a);
        (*launches)++;
    } while (at < count);
    return cudaGetLastError();
}

}  // namespace

// Two table sizes: the parameters of a launch are copied with it.
constexpr int SMALL_CAP = 64, NORM_CAP = 1024, ADAM_CAP = 512;

cudaError_t launch_clip(cudaStream_t st, int count, float* const* grads, const long long* sizes, float max_norm, float eps,
                        bool scale, float* norm_out, float* coef_out, void* workspace, unsigned int* ticket, int num_sms,
                        long long* launches)
{
    if (count <= SMALL_CAP)
        return clip_cap<SMALL_CAP>(st, count, grads, sizes, max_norm, eps, scale, norm_out, coef_out, workspace, ticket, num_sms, launches);
    return clip_cap<NORM_CAP>(st, count, grads, sizes, max_norm, eps, scale, norm_out, coef_out, workspace, ticket, num_sms, launches);
}

cudaError_t launch_adam(cudaStream_t st, int count, float* const* p, const float* const* g, float* const* m,
                        float* const* v, const long long* sizes, float* adv, const float* grad_scale, float b1, float b2,
                        float lr, float eps, float cwd, float dfac, bool advance, unsigned int* ticket, int num_sms,
                        long long* launches)
{
    const AdamArgs a{adv, grad_scale, b1, b2, lr, eps, cwd, dfac, advance ? 1 : 0, 1, ticket};
    if (count <= SMALL_CAP) return adam_cap<SMALL_CAP>(st, count, p, g, m, v, sizes, a, num_sms, launches);
    return adam_cap<ADAM_CAP>(st, count, p, g, m, v, sizes, a, num_sms, launches);
}

}  // namespace lists
}  // namespace tt
