// Global norm of many gradients, and clipping.
//
//   norm = (sum g^2)^(1/2) over all tensors (or max |g|),  f = min(1, max_norm / (norm + 1e-6)),  dst = f * src
//
// Two passes over the data, bound by memory: the norm reads every element once, the second pass reads and writes it.  Both
// split every tensor into chunks of CHUNK elements and hand the chunks of ALL tensors to one grid, so that the number of
// launches depends on the number of tensors (128 in a launch's argument block), not on their sizes, and no table of addresses
// has to be copied to the device (a captured graph holds the arguments itself).
// Squares are summed in 64 bits: fp32 squares overflow from 1.8e19 on and underflow below 1e-23, and the conversion is free
// beside the loads.  Every workgroup leaves one partial sum; the second pass adds the partial sums again in every workgroup, in
// one fixed order, instead of a launch between the two: up to DIRECT of them (16 KB from the L2 cache).
// Measured, 2^30 bf16 elements in 60 tensors: norm 369 us (5.8 TB/s), scaling 802 (5.4 TB/s; a copy of 2 GB runs at 4.7); 57 fp32
// tensors of a generator, 52 MB: 12 and 20 us (4.2, 5.2 TB/s), less than the host takes to hand over the list.
// Without a tensor whose dst differs from src, the second pass ends at once where the factor is 1.
#include "text_common.h"

namespace {
using namespace s2ag;
using namespace s2ag::text;

constexpr int GROUP = 128;              // tensors of a launch: 128 * 28 + 8 bytes of arguments, under the 4 KB there are
constexpr int CHUNK = 16384;            // elements
constexpr int MAX_BLOCKS = 1024;        // four workgroups of 256 threads on each of 256 compute units
constexpr int DIRECT = 2048;

struct Table {
    const void* src[GROUP];
    void* dst[GROUP];
    long long n[GROUP];                 // elements; bit 62: src is bf16, bit 61: dst is bf16
    unsigned first[GROUP + 1];          // chunk number of the tensor's first chunk
    int tensors;
};
static_assert(sizeof(Table) <= 3712, "kernel argument block");
constexpr long long SRC16 = 1LL << 62, DST16 = 1LL << 61, COUNT = DST16 - 1;

__device__ __forceinline__ int tensor_of(const Table& t, unsigned chunk) {
    int lo = 0, hi = t.tensors - 1;     // the last tensor whose first chunk is not behind `chunk` (empty tensors have none)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// fixed order: lanes by halving, then the wavefronts in turn
template <bool INF> __device__ __forceinline__ double join(double a, double b) {
    if (!INF) return a + b;
    if (a != a) return a;               // a NaN stays
    return (b != b || b > a) ? b : a;
}
template <bool INF> __device__ double block_join(double v, double* sm) {
    for (int d = 32; d >= 1; d >>= 1) v = join<INF>(v, __shfl_xor(v, d));
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[wave] = v;
    __syncthreads();
    double s = sm[0];
    for (int w = 1; w < waves; ++w) s = join<INF>(s, sm[w]);
    return s;
}

template <bool INF> __device__ __forceinline__ double take(double s, float g) {
    const double v = (double)g;
    return INF ? join<true>(s, fabs(v)) : s + v * v;
}

template <bool INF, typename T>
__device__ double chunk_sum(const T* __restrict__ p, int n) {
    constexpr int V = Vec<T>::N;
    double s0 = 0.0, s1 = 0.0;
    int i = threadIdx.x * V;
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        for (; i + 3 * 256 * V + V <= n; i += 4 * 256 * V) {      // four loads in flight
            float v[4][V];
            for (int u = 0; u < 4; ++u) Vec<T>::load(p + i + u * 256 * V, v[u]);
            for (int u = 0; u < 4; ++u)
                for (int j = 0; j < V; j += 2) {
                    s0 = take<INF>(s0, v[u][j]);
                    s1 = take<INF>(s1, v[u][j + 1]);
                }
        }
        for (; i + V <= n; i += 256 * V) {
            float v[V];
            Vec<T>::load(p + i, v);
            for (int j = 0; j < V; ++j) s0 = take<INF>(s0, v[j]);
        }
        for (int j = n - n % V + threadIdx.x; j < n; j += 256) s1 = take<INF>(s1, (float)p[j]);
    } else {
        for (int j = threadIdx.x; j < n; j += 256) s0 = take<INF>(s0, (float)p[j]);
    }
    return join<INF>(s0, s1);
}

template <bool INF>
__global__ __launch_bounds__(256) void norm_k(Table t, double* __restrict__ partials) {
    __shared__ double sm[4];
    double s = 0.0;
    const unsigned chunks = t.first[t.tensors];
    for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int k = tensor_of(t, c);
        const long long off = (long long)(c - t.first[k]) * CHUNK, left = (t.n[k] & COUNT) - off;
        const int n = left < CHUNK ? (int)left : CHUNK;
        const double v = (t.n[k] & SRC16) ? chunk_sum<INF>(static_cast<const bf16_t*>(t.src[k]) + off, n)
                                          : chunk_sum<INF>(static_cast<const float*>(t.src[k]) + off, n);
        s = join<INF>(s, v);
    }
    s = block_join<INF>(s, sm);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

template <bool INF> __device__ double sum_partials(const double* __restrict__ partials, int count, double* sm) {
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += 256) s = join<INF>(s, partials[i]);
    return block_join<INF>(s, sm);
}

template <bool INF>
__global__ __launch_bounds__(256) void fold_k(double* partials, int count) {
    __shared__ double sm[4];
    const double s = sum_partials<INF>(partials, count, sm);       // (every thread has read its share: block_join waits)
    if (threadIdx.x == 0) partials[0] = s;
}

template <typename S, typename D>
__device__ void chunk_scale(const S* src, D* dst, int n, float f) {
    constexpr int V = 8;
    if (((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 15) == 0) {
        int i = threadIdx.x * V;
        for (; i + 256 * V + V <= n; i += 2 * 256 * V) {
            float v[2][V];
            for (int u = 0; u < 2; ++u)
                for (int j = 0; j < V; j += Vec<S>::N) Vec<S>::load(src + i + u * 256 * V + j, v[u] + j);
            for (int u = 0; u < 2; ++u) {
                for (int j = 0; j < V; ++j) v[u][j] *= f;
                for (int j = 0; j < V; j += Vec<D>::N) Vec<D>::store(dst + i + u * 256 * V + j, v[u] + j);
            }
        }
        for (; i + V <= n; i += 256 * V) {
            float v[V];
            for (int j = 0; j < V; j += Vec<S>::N) Vec<S>::load(src + i + j, v + j);
            for (int j = 0; j < V; ++j) v[j] *= f;
            for (int j = 0; j < V; j += Vec<D>::N) Vec<D>::store(dst + i + j, v + j);
        }
        for (int j = n - n % V + threadIdx.x; j < n; j += 256) dst[j] = (D)((float)src[j] * f);
    } else {
        for (int j = threadIdx.x; j < n; j += 256) dst[j] = (D)((float)src[j] * f);
    }
}

template <bool INF>
__global__ __launch_bounds__(256) void scale_k(Table t, const double* __restrict__ partials, int count, float max_norm,
                                               float* __restrict__ norm_out) {
    __shared__ double sm[4];
    const double s = sum_partials<INF>(partials, count, sm);
    const float norm = (float)(INF ? s : sqrt(s));
    float f = max_norm / (norm + 1e-6f);
    f = f > 1.f ? 1.f : f;                                        // (NaN stays NaN)
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    const unsigned chunks = t.first[t.tensors];
    // backwards: what the norm read last is still in the memory-side cache
    for (unsigned i = blockIdx.x; i < chunks; i += gridDim.x) {
        const unsigned c = chunks - 1 - i;
        const int k = tensor_of(t, c);
        if (!t.dst[k] || (f == 1.f && t.dst[k] == t.src[k])) continue;
        const long long off = (long long)(c - t.first[k]) * CHUNK, left = (t.n[k] & COUNT) - off;
        const int n = left < CHUNK ? (int)left : CHUNK;
        const bool s16 = t.n[k] & SRC16, d16 = t.n[k] & DST16;
        if (s16 && d16) chunk_scale(static_cast<const bf16_t*>(t.src[k]) + off, static_cast<bf16_t*>(t.dst[k]) + off, n, f);
        else if (s16) chunk_scale(static_cast<const bf16_t*>(t.src[k]) + off, static_cast<float*>(t.dst[k]) + off, n, f);
        else if (d16) chunk_scale(static_cast<const float*>(t.src[k]) + off, static_cast<bf16_t*>(t.dst[k]) + off, n, f);
        else chunk_scale(static_cast<const float*>(t.src[k]) + off, static_cast<float*>(t.dst[k]) + off, n, f);
    }
}

// fills the table with the tensors from `at` on; returns the chunk count
unsigned fill(Table& t, const s2ag_clip_tensor* a, int at, int tensors) {
    t.tensors = tensors - at < GROUP ? tensors - at : GROUP;
    unsigned chunks = 0;
    for (int i = 0; i < t.tensors; ++i) {
        const s2ag_clip_tensor& q = a[at + i];
        t.src[i] = q.src;
        t.dst[i] = q.dst;
        t.n[i] = q.n | (q.src_bf16 ? SRC16 : 0) | (q.dst_bf16 ? DST16 : 0);
        t.first[i] = chunks;
        chunks += (unsigned)((q.n + CHUNK - 1) / CHUNK);
    }
    t.first[t.tensors] = chunks;
    return chunks;
}

int blocks_of(unsigned chunks) { return chunks < 1 ? 1 : chunks < (unsigned)MAX_BLOCKS ? (int)chunks : MAX_BLOCKS; }

bool valid(const s2ag_clip_tensor* a, int tensors) {
    if (tensors < 0 || (tensors && !a)) return false;
    // 2^38 elements are 2^24 chunks of 2^14; a launch's 128 tensors have 2^31 at most, which an unsigned holds
    for (int i = 0; i < tensors; ++i)
        if (a[i].n < 0 || a[i].n > (1LL << 38) || (a[i].n && !a[i].src)) return false;
    return true;
}

template <bool INF>
int run(const s2ag_clip_tensor* a, int tensors, float max_norm, double* partials, float* norm, hipStream_t st) {
    Table t;
    int count = 0;
    int at = 0;
    do {                                                          // (no tensors: one workgroup writes a norm of 0)
        const int g = blocks_of(fill(t, a, at, tensors));
        hipLaunchKernelGGL(norm_k<INF>, dim3(g), dim3(256), 0, st, t, partials + count);
        S2AG_LAUNCH_CHECK();
        count += g;
        at += GROUP;
    } while (at < tensors);
    if (count > DIRECT) {
        hipLaunchKernelGGL(fold_k<INF>, dim3(1), dim3(256), 0, st, partials, count);
        S2AG_LAUNCH_CHECK();
        count = 1;
    }
    float* out = norm;
    at = tensors > 0 ? (tensors - 1) / GROUP * GROUP : 0;
    do {
        const unsigned chunks = fill(t, a, at, tensors);
        bool write = false;
        for (int i = 0; i < t.tensors; ++i) write |= t.dst[i] != nullptr;
        if (write || out) {
            if (!write) t.first[t.tensors] = 0;
            hipLaunchKernelGGL(scale_k<INF>, dim3(write ? blocks_of(chunks) : 1), dim3(256), 0, st, t, partials, count, max_norm, out);
            S2AG_LAUNCH_CHECK();
        }
        out = nullptr;
        at -= GROUP;
    } while (at >= 0);
    return 0;
}
}  // namespace

extern "C" long long s2ag_clip_partials(const s2ag_clip_tensor* t, int tensors) {
    if (!valid(t, tensors)) return S2AG_E_BADARG;
    Table tab;
    long long count = 0;
    int at = 0;
    do {
        count += blocks_of(fill(tab, t, at, tensors));
        at += GROUP;
    } while (at < tensors);
    return count;
}

extern "C" int s2ag_clip_grads(const s2ag_clip_tensor* t, int tensors, float max_norm, int norm_inf, double* partials, float* norm,
                               void* stream) {
    if (!valid(t, tensors) || !partials || !norm || !(max_norm >= 0.f)) return S2AG_E_BADARG;
    for (int i = 0; i < tensors; ++i)
        if (t[i].src == t[i].dst && t[i].src_bf16 != t[i].dst_bf16) return S2AG_E_BADARG;
    return norm_inf ? run<true>(t, tensors, max_norm, partials, norm, (hipStream_t)stream)
                    : run<false>(t, tensors, max_norm, partials, norm, (hipStream_t)stream);
}
