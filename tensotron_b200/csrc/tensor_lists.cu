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
constexpr int SMALL_THREADS = 1024, SMALL_CHUNK = 512;
constexpr long long SMALL_ELEMENTS = 32768; // lists up to this many elements are clipped by one CTA
// The last chunks of a list, which the launch behind the norm reads first, are read into L2's long-lived lines; the others
// pass by.
constexpr int KEEP_CHUNKS = (80 << 20) / (CHUNK * 4);

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

// The tensor that chunk `c` belongs to: the last one whose first chunk is at most c.  The search starts where a list of equal
// tensors has it (256 equal tensors: 6.1 us for the norm instead of 6.7, the table's words come one after the other).
template <typename T>
__device__ __forceinline__ int tensor_of(const T& t, int c)
{
    int lo = 0, hi = t.count;
    const int guess = min(t.count - 1, static_cast<int>(static_cast<float>(c) * (static_cast<float>(t.count) / static_cast<float>(t.chunks))));
    const int at = t.first[guess], behind = t.first[guess + 1];
    if (c < at) hi = guess;
    else if (c < behind) return guess;
    else lo = guess + 1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= c) lo = mid; else hi = mid;
    }
    return lo;
}

// Chunk `c` of CH elements of a tensor of `size` elements whose first `head` elements lie in front of the 16-byte boundary,
// walked by NT threads of which the caller is number `t`: body1(i) for the elements outside aligned groups of four,
// body4(i, n) for up to CH / 4 / NT such groups at i, i + 4 NT, ... of which the first n exist, so that a thread asks for all of
// its elements before it uses the first.
template <int CH, int NT, typename F4, typename F1>
__device__ __forceinline__ void for_chunk(int c, long long size, int head, int t, F4 body4, F1 body1)
{
    constexpr int G = CH / 4 / NT;
    const long long lo = head + static_cast<long long>(c) * CH;
    const long long hi = lo + CH < size ? lo + CH : size;
    if (c == 0 && t < head && t < size) body1(static_cast<long long>(t));
    const int n4 = hi > lo ? static_cast<int>((hi - lo) >> 2) : 0;
    const int n = n4 >= CH / 4 ? G : n4 > t ? (n4 - t + NT - 1) / NT : 0;
    if (n > 0) body4(lo + 4ll * t, n);
    const long long tail = lo + 4ll * n4 + t;
    if (t < 4 && tail < hi) body1(tail);
}

constexpr int GROUPS = CHUNK / 4 / THREADS;          // 128-bit pieces of a full chunk per thread

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

// As for the adapters' launches: the norm lets the launch behind it begin, which waits before it reads anything.
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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
// sums in a fixed order.  36.8 M elements: 27 us cold (147 MB: 22.5 at the copy rate), 31-33 behind a launch whose stores are still
// on their way to memory; float sums take the same time.
template <int CAP>
__global__ void __launch_bounds__(THREADS) norm_kernel(const __grid_constant__ NormTable<CAP> t, const NormFinish f)
{
    __shared__ double red[THREADS / 32];
    __shared__ unsigned int last;
    let_next_begin();
    double s = 0.0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const float* g = t.ptr[i];
        const bool keep = c >= t.chunks - KEEP_CHUNKS;
        for_chunk<CHUNK, THREADS>(c - t.first[i], t.size[i], head_of(g), threadIdx.x,
                  [&](long long e, int n) {
                      const float4* src = reinterpret_cast<const float4*>(g + e);
                      float4 v[GROUPS];
                      if (keep) {
#pragma unroll
                          for (int k = 0; k < GROUPS; k++) v[k] = k < n ? src[THREADS * k] : make_float4(0.f, 0.f, 0.f, 0.f);
                      } else {
#pragma unroll
                          for (int k = 0; k < GROUPS; k++) v[k] = k < n ? __ldcs(src + THREADS * k) : make_float4(0.f, 0.f, 0.f, 0.f);
                      }
#pragma unroll
                      for (int k = 0; k < GROUPS; k++) s += (square(v[k].x) + square(v[k].y)) + (square(v[k].z) + square(v[k].w));
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

// (from the last chunk to the first: what the norm read last is still in L2: 101 of 147 MB come from memory, 43 us; norm and
// scaling together move 395 MB in 72 us)
template <int CAP>
__global__ void __launch_bounds__(THREADS) scale_kernel(const __grid_constant__ NormTable<CAP> t, const float* coef_ptr)
{
    wait_for_previous();
    const float coef = __ldcg(coef_ptr);
    for (int c = t.chunks - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
        const int i = tensor_of(t, c);
        float* g = t.ptr[i];
        for_chunk<CHUNK, THREADS>(c - t.first[i], t.size[i], head_of(g), threadIdx.x,
                  [&](long long e, int n) {
                      float4 v[GROUPS];
#pragma unroll
                      for (int k = 0; k < GROUPS; k++)
                          if (k < n) v[k] = __ldcs(reinterpret_cast<const float4*>(g + e + 4ll * THREADS * k));
#pragma unroll
                      for (int k = 0; k < GROUPS; k++)
                          if (k < n) __stcs(reinterpret_cast<float4*>(g + e + 4ll * THREADS * k), make_float4(v[k].x * coef, v[k].y * coef, v[k].z * coef, v[k].w * coef));
                  },
                  [&](long long e) { g[e] *= coef; });
    }
}

// A short list in one launch of one CTA: its warps share out chunks of SMALL_CHUNK elements, and what they scale they have
// just read.
template <int CAP>
__global__ void __launch_bounds__(SMALL_THREADS) clip_small_kernel(const __grid_constant__ NormTable<CAP> t, float max_norm, float eps, int scale,
                                                                   float* norm_out, float* coef_out)
{
    __shared__ double red[SMALL_THREADS / 32];
    let_next_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int G = SMALL_CHUNK / 4 / 32;
    double s = 0.0;
    for (int c = warp; c < t.chunks; c += SMALL_THREADS / 32) {
        const int i = tensor_of(t, c);
        const float* g = t.ptr[i];
        for_chunk<SMALL_CHUNK, 32>(c - t.first[i], t.size[i], head_of(g), lane,
                  [&](long long e, int n) {
                      float4 v[G];
#pragma unroll
                      for (int k = 0; k < G; k++) v[k] = k < n ? *reinterpret_cast<const float4*>(g + e + 128 * k) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                      for (int k = 0; k < G; k++) s += (square(v[k].x) + square(v[k].y)) + (square(v[k].z) + square(v[k].w));
                  },
                  [&](long long e) { s += square(g[e]); });
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    s = 0.0;
    for (int w = 0; w < SMALL_THREADS / 32; w++) s += red[w];
    const float norm = static_cast<float>(sqrt(s)), coef = clip_coef(norm, max_norm, eps);
    if (threadIdx.x == 0) {
        if (norm_out) *norm_out = norm;
        if (coef_out) *coef_out = coef;
    }
    if (!scale) return;
    for (int c = warp; c < t.chunks; c += SMALL_THREADS / 32) {
        const int i = tensor_of(t, c);
        float* g = t.ptr[i];
        for_chunk<SMALL_CHUNK, 32>(c - t.first[i], t.size[i], head_of(g), lane,
                  [&](long long e, int n) {
#pragma unroll
                      for (int k = 0; k < G; k++)
                          if (k < n) {
                              float4 v = *reinterpret_cast<const float4*>(g + e + 128 * k);
                              v.x *= coef; v.y *= coef; v.z *= coef; v.w *= coef;
                              *reinterpret_cast<float4*>(g + e + 128 * k) = v;
                          }
                  },
                  [&](long long e) { g[e] *= coef; });
    }
}

// 28 bytes per element: 36.8 M elements in 169 us (1030 MB: 158 at the copy rate).
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
    wait_for_previous();
    if (threadIdx.x == 0) {
        if (a.advance) {
            const float step = __ldcg(a.adv) + 1.f;
            fix[0] = step;
            fix[1] = 1.f / (1.f - powf(a.b1, step));
            fix[2] = 1.f / (1.f - powf(a.b2, step));
        } else {
            fix[1] = __ldcg(a.adv + 1);
            fix[2] = __ldcg(a.adv + 2);
        }
    }
    __syncthreads();
    const float ibc1 = fix[1], ibc2 = fix[2], omb1 = 1.f - a.b1, omb2 = 1.f - a.b2;
    const float coef = a.grad_scale ? __ldcg(a.grad_scale) : 1.f;
    // The scaled gradient is rounded (not contracted into what follows), as if it had been clipped in place.
    // (from the last chunk to the first, and p, m and v past the L2's long-lived lines: gradients that a norm has just read
    // are still there)
    for (int c = t.chunks - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
        const int i = tensor_of(t, c);
        float* p = t.p[i];
        const float* g = t.g[i];
        float* m = t.m[i];
        float* v = t.v[i];
        const int head = head_of(p);
        const bool vec = head_of(g) == head && head_of(m) == head && head_of(v) == head;
        const auto one = [&](long long e) {
            float pp = p[e], mm = m[e], vv = v[e];
            ew::adam_one(pp, __fmul_rn(coef, g[e]), mm, vv, a.b1, omb1, a.b2, omb2, a.lr, a.eps, ibc1, ibc2, a.cwd, a.dfac);
            p[e] = pp; m[e] = mm; v[e] = vv;
        };
        if (!vec) {
            // the four tensors of this parameter start at different places behind a 16-byte boundary
            const long long lo = static_cast<long long>(c - t.first[i]) * CHUNK, hi = lo + CHUNK < t.size[i] ? lo + CHUNK : t.size[i];
            for (long long e = lo + threadIdx.x; e < hi; e += THREADS) one(e);
            continue;
        }
        for_chunk<CHUNK, THREADS>(c - t.first[i], t.size[i], head, threadIdx.x,
                  [&](long long e0, int n) {
#pragma unroll
                      for (int k0 = 0; k0 < GROUPS; k0 += 2) {
                          float4 pp[2], gg[2], mm[2], vv[2];
#pragma unroll
                          for (int k = 0; k < 2; k++) {
                              const long long e = e0 + 4ll * THREADS * (k0 + k);
                              if (k0 + k >= n) continue;
                              pp[k] = __ldcs(reinterpret_cast<const float4*>(p + e));
                              gg[k] = *reinterpret_cast<const float4*>(g + e);
                              mm[k] = __ldcs(reinterpret_cast<const float4*>(m + e));
                              vv[k] = __ldcs(reinterpret_cast<const float4*>(v + e));
                          }
#pragma unroll
                          for (int k = 0; k < 2; k++) {
                              const long long e = e0 + 4ll * THREADS * (k0 + k);
                              if (k0 + k >= n) continue;
                              ew::adam_one(pp[k].x, __fmul_rn(coef, gg[k].x), mm[k].x, vv[k].x, a.b1, omb1, a.b2, omb2, a.lr, a.eps, ibc1, ibc2, a.cwd, a.dfac);
                              ew::adam_one(pp[k].y, __fmul_rn(coef, gg[k].y), mm[k].y, vv[k].y, a.b1, omb1, a.b2, omb2, a.lr, a.eps, ibc1, ibc2, a.cwd, a.dfac);
                              ew::adam_one(pp[k].z, __fmul_rn(coef, gg[k].z), mm[k].z, vv[k].z, a.b1, omb1, a.b2, omb2, a.lr, a.eps, ibc1, ibc2, a.cwd, a.dfac);
                              ew::adam_one(pp[k].w, __fmul_rn(coef, gg[k].w), mm[k].w, vv[k].w, a.b1, omb1, a.b2, omb2, a.lr, a.eps, ibc1, ibc2, a.cwd, a.dfac);
                              __stcs(reinterpret_cast<float4*>(p + e), pp[k]);
                              __stcs(reinterpret_cast<float4*>(m + e), mm[k]);
                              __stcs(reinterpret_cast<float4*>(v + e), vv[k]);
                          }
                      }
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

long long chunks_of(long long size, int head, int chunk)
{
    const long long body = size - head;
    return size <= 0 ? 0 : body <= 0 ? 1 : (body + chunk - 1) / chunk;
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
bool fill(NormTable<CAP>& t, int count, float* const* ptr, const long long* sizes, int* at, int chunk = CHUNK)
{
    t.count = t.chunks = 0;
    for (; *at < count && t.count < CAP; (*at)++) {
        const long long n = chunks_of(sizes[*at], head_of(ptr[*at]), chunk);
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

// Launches a kernel that waits, before it reads anything, for the launch in front of it, and may begin while that one ends.
template <typename... P>
cudaError_t launch_early(cudaStream_t st, void (*kernel)(P...), int grid, const P&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
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
    long long elements = 0;
    for (int i = 0; i < count && elements <= SMALL_ELEMENTS; i++) elements += sizes[i];
    if (count <= CAP && elements <= SMALL_ELEMENTS) {
        // 8-64-64-2 (six tensors): 3.4 us on the GPU against 3.4 + 2.0 in two launches
        fill(t, count, grads, sizes, &at, SMALL_CHUNK);
        clip_small_kernel<CAP><<<1, SMALL_THREADS, 0, st>>>(t, max_norm, eps, scale ? 1 : 0, norm_out, coef_out);
        (*launches)++;
        return cudaGetLastError();
    }
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
            const cudaError_t e = launch_early(st, scale_kernel<CAP>, grid_of(t.chunks, num_sms), t, static_cast<const float*>(coef));
            if (e != cudaSuccess) return e;
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
            const long long n = chunks_of(sizes[at], vec ? head : 0, CHUNK);
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
        const cudaError_t e = launch_early(st, adam_kernel<CAP>, grid_of(t.chunks, num_sms), t, a);
        if (e != cudaSuccess) return e;
        (*launches)++;
    } while (at < count);
    return cudaGetLastError();
}

}  // namespace

// Table sizes: the parameters of a launch are copied with it (20 and 44 bytes per tensor).
constexpr int SMALL_CAP = 64, MID_CAP = 320, NORM_CAP = 1024, ADAM_CAP = 640;

cudaError_t launch_clip(cudaStream_t st, int count, float* const* grads, const long long* sizes, float max_norm, float eps,
                        bool scale, float* norm_out, float* coef_out, void* workspace, unsigned int* ticket, int num_sms,
                        long long* launches)
{
    if (count <= SMALL_CAP)
        return clip_cap<SMALL_CAP>(st, count, grads, sizes, max_norm, eps, scale, norm_out, coef_out, workspace, ticket, num_sms, launches);
    if (count <= MID_CAP)
        return clip_cap<MID_CAP>(st, count, grads, sizes, max_norm, eps, scale, norm_out, coef_out, workspace, ticket, num_sms, launches);
    return clip_cap<NORM_CAP>(st, count, grads, sizes, max_norm, eps, scale, norm_out, coef_out, workspace, ticket, num_sms, launches);
}

cudaError_t launch_adam(cudaStream_t st, int count, float* const* p, const float* const* g, float* const* m,
                        float* const* v, const long long* sizes, float* adv, const float* grad_scale, float b1, float b2,
                        float lr, float eps, float cwd, float dfac, bool advance, unsigned int* ticket, int num_sms,
                        long long* launches)
{
    const AdamArgs a{adv, grad_scale, b1, b2, lr, eps, cwd, dfac, advance ? 1 : 0, 1, ticket};
    if (count <= SMALL_CAP) return adam_cap<SMALL_CAP>(st, count, p, g, m, v, sizes, a, num_sms, launches);
    if (count <= MID_CAP) return adam_cap<MID_CAP>(st, count, p, g, m, v, sizes, a, num_sms, launches);
    return adam_cap<ADAM_CAP>(st, count, p, g, m, v, sizes, a, num_sms, launches);
}

namespace {
template <int CAP>
cudaError_t load_norm()
{
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, norm_kernel<CAP>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, scale_kernel<CAP>);
    return e != cudaSuccess ? e : cudaFuncGetAttributes(&attr, clip_small_kernel<CAP>);
}

template <int CAP>
cudaError_t load_adam()
{
    cudaFuncAttributes attr;
    return cudaFuncGetAttributes(&attr, adam_kernel<CAP>);
}
}  // namespace

cudaError_t init_lists()
{
    cudaError_t e;
    if ((e = load_norm<SMALL_CAP>()) != cudaSuccess || (e = load_norm<MID_CAP>()) != cudaSuccess || (e = load_norm<NORM_CAP>()) != cudaSuccess ||
        (e = load_adam<SMALL_CAP>()) != cudaSuccess || (e = load_adam<MID_CAP>()) != cudaSuccess)
        return e;
    return load_adam<ADAM_CAP>();
}

}  // namespace lists
}  // namespace tt
