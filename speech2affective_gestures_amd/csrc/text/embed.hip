// Embedding lookup with a scale, and its gradient by sorted ids.
//
//   out_i = scale * T[id_i]                 dT_v = scale * sum_{i : id_i = v} dy_i
//
// Both are bound by memory.  The gradient sorts (id, position) pairs with a stable radix sort, so that the rows of one id are
// neighbours IN THE ORDER OF THEIR POSITIONS, and sums each run of equal ids in registers in that order: no atomics, the same
// bits every time.  Text has a few ids with very many positions (padding, frequent words) and many with one, so the sorted list
// is cut into tiles of equal length, not by id: a wavefront sums TILE positions of 64 * V columns, writes the runs that lie
// inside its tile, and leaves the sums of the runs that cross a tile's border (at most two a tile) to a second launch, which
// adds the pieces of a run in order.
//
// ids that are not in the table, and the padding row's, sort behind the last row under the key n_entries and are not summed.
#include "text_common.h"

namespace {
using namespace s2ag;
using namespace s2ag::text;

// ---- lookup ----------------------------------------------------------------------------------------------------------------
// A row is read by 2^tx_log lanes, 16 bytes each where every row starts at a multiple of 16 bytes.
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256) void lookup_k(const void* __restrict__ ids, int ids_i32, const T* __restrict__ table, long long n,
                                                int dim, long long n_entries, float scale, T* __restrict__ out, int tx_log) {
    constexpr int V = ALIGNED ? Vec<T>::N : 1;
    const int tx = threadIdx.x & ((1 << tx_log) - 1), ty = threadIdx.x >> tx_log, rows = 256 >> tx_log;
    for (long long r = (long long)blockIdx.x * rows + ty; r < n; r += (long long)gridDim.x * rows) {
        const long long id = load_id(ids, ids_i32, r);
        const bool in = id >= 0 && id < n_entries;
        const T* src = table + (in ? id : 0) * dim;
        T* dst = out + r * dim;
        for (int c = tx * V; c < dim; c += V << tx_log) {
            if constexpr (ALIGNED) {
                float v[V];
                Vec<T>::load(src + c, v);
                for (int j = 0; j < V; ++j) v[j] = in ? v[j] * scale : 0.f;
                Vec<T>::store(dst + c, v);
            } else {
                dst[c] = in ? (T)((float)src[c] * scale) : (T)0.f;
            }
        }
    }
}

// ---- stable radix sort -----------------------------------------------------------------------------------------------------
// Among the lanes of a wavefront: how many lower lanes hold the same digit, and whether this is the highest of them.
template <int BITS>
__device__ __forceinline__ int lower_peers(unsigned digit, int lane, int* total) {
    unsigned long long peers = ~0ULL;
    for (int b = 0; b < BITS; ++b) {
        const unsigned long long m = __ballot((digit >> b) & 1);
        peers &= ((digit >> b) & 1) ? m : ~m;
    }
    *total = __popcll(peers);
    return __popcll(peers & ((1ULL << lane) - 1));
}

// Inclusive sum over the `lanes` (a power of two) first lanes.
__device__ __forceinline__ int wave_scan(int v, int lane) {
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d);
        if (lane >= d) v += u;
    }
    return v;
}

__device__ __forceinline__ unsigned key_of(const void* ids, int ids_i32, long long i, long long n_entries, long long padding_idx) {
    const long long id = load_id(ids, ids_i32, i);
    return (unsigned)((id < 0 || id >= n_entries || id == padding_idx) ? n_entries : id);
}

// Up to SMALL positions: one workgroup sorts them in LDS, 8 bits a pass.  Items go by wavefront, round and lane, which is their
// order; a wavefront counts its items per digit while it ranks them, so that a pass reads its items once.
constexpr int SMALL = 8192;
constexpr int SB = 8, SBINS = 1 << SB, SWAVES = 16, SROUNDS = SMALL / 1024;
__global__ __launch_bounds__(1024) void sort_small_k(const void* __restrict__ ids, int ids_i32, int n, long long n_entries,
                                                     long long padding_idx, int passes, int clear_flags,
                                                     unsigned* __restrict__ keys, int* __restrict__ pos,
                                                     unsigned char* __restrict__ touched) {
    __shared__ unsigned k_s[SMALL];
    __shared__ unsigned short p_s[SMALL];
    __shared__ unsigned short cnt[SWAVES][SBINS];
    __shared__ int base[SBINS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (touched && clear_flags)
        for (long long i = tid; i < n_entries; i += 1024) touched[i] = 0;
    const int items = wave * (SROUNDS * 64) + lane;
    unsigned key[SROUNDS];
    int at[SROUNDS], rank[SROUNDS];
    for (int r = 0; r < SROUNDS; ++r) {
        const int i = items + r * 64;
        at[r] = i;
        key[r] = i < n ? key_of(ids, ids_i32, i, n_entries, padding_idx) : ~0u;     // behind every key there is
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * SB;
        for (int i = tid; i < SWAVES * SBINS; i += 1024) (&cnt[0][0])[i] = 0;
        __syncthreads();
        for (int r = 0; r < SROUNDS; ++r) {
            const unsigned d = (key[r] >> shift) & (SBINS - 1);
            int total;
            const int low = lower_peers<SB>(d, lane, &total);
            const int before = cnt[wave][d];
            __builtin_amdgcn_wave_barrier();
            rank[r] = before + low;
            if (low == total - 1) cnt[wave][d] = (unsigned short)(before + total);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        if (tid < SBINS) {
            int s = 0;
            for (int w = 0; w < SWAVES; ++w) {
                const int c = cnt[w][tid];
                cnt[w][tid] = (unsigned short)s;
                s += c;
            }
            base[tid] = s;
        }
        __syncthreads();
        if (wave == 0) {                                         // exclusive sums over the digits, four to a lane
            int v[4], s = 0;
            for (int j = 0; j < 4; ++j) {
                v[j] = base[lane * 4 + j];
                s += v[j];
            }
            int e = wave_scan(s, lane) - s;
            for (int j = 0; j < 4; ++j) {
                base[lane * 4 + j] = e;
                e += v[j];
            }
        }
        __syncthreads();
        for (int r = 0; r < SROUNDS; ++r) {
            const unsigned d = (key[r] >> shift) & (SBINS - 1);
            const int to = base[d] + cnt[wave][d] + rank[r];
            k_s[to] = key[r];
            p_s[to] = (unsigned short)at[r];
        }
        __syncthreads();
        for (int r = 0; r < SROUNDS; ++r) {
            key[r] = k_s[items + r * 64];
            at[r] = p_s[items + r * 64];
        }
        __syncthreads();
    }
    for (int r = 0; r < SROUNDS; ++r) {
        const int i = items + r * 64;
        if (i < n) {
            keys[i] = key[r];
            pos[i] = at[r];
            if (touched && key[r] < (unsigned)n_entries) touched[key[r]] = 1;
        }
    }
}

// More: per pass of LB bits one launch counts the digits of every tile of LTILE items, one adds the counts up over the tiles
// (a workgroup per digit), one moves the items.
constexpr int LB = 9, LBINS = 1 << LB, LTILE = 4096, LWAVES = 4, LROUNDS = LTILE / 256;
struct SortIn {
    const void* ids;                    // first pass: the keys come from the ids, the positions count up
    int ids_i32;
    long long n_entries, padding_idx;
    const unsigned* keys;
    const int* pos;
    int n;
};
__device__ __forceinline__ unsigned sort_key(const SortIn& in, int i) {
    return in.ids ? key_of(in.ids, in.ids_i32, i, in.n_entries, in.padding_idx) : in.keys[i];
}

__global__ __launch_bounds__(256) void sort_count_k(SortIn in, int shift, int tiles, int* __restrict__ counts) {
    __shared__ int c[LBINS];
    for (int i = threadIdx.x; i < LBINS; i += 256) c[i] = 0;
    __syncthreads();
    const int t0 = blockIdx.x * LTILE;
    for (int r = 0; r < LROUNDS; ++r) {
        const int i = t0 + r * 256 + threadIdx.x;
        if (i < in.n) atomicAdd(&c[(sort_key(in, i) >> shift) & (LBINS - 1)], 1);     // (whole numbers: any order, one sum)
    }
    __syncthreads();
    for (int i = threadIdx.x; i < LBINS; i += 256) counts[(long long)i * tiles + blockIdx.x] = c[i];
}

__global__ __launch_bounds__(256) void sort_scan_k(int tiles, int* __restrict__ counts, int* __restrict__ totals) {
    __shared__ int sm[4];
    int* c = counts + (long long)blockIdx.x * tiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int carry = 0;
    for (int t0 = 0; t0 < tiles; t0 += 256) {
        const int t = t0 + threadIdx.x, v = t < tiles ? c[t] : 0;
        const int inc = wave_scan(v, lane);
        if (lane == 63) sm[wave] = inc;
        __syncthreads();
        int add = carry;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) add += sm[w];
            carry += sm[w];
        }
        if (t < tiles) c[t] = add + inc - v;
        __syncthreads();
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

__global__ __launch_bounds__(256) void sort_move_k(SortIn in, int shift, int tiles, const int* __restrict__ counts,
                                                   const int* __restrict__ totals, unsigned* __restrict__ keys_out,
                                                   int* __restrict__ pos_out, unsigned char* __restrict__ touched) {
    __shared__ unsigned short cnt[LWAVES][LBINS];
    __shared__ int base[LBINS];
    __shared__ int sm[LWAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < LWAVES * LBINS; i += 256) (&cnt[0][0])[i] = 0;
    // where each digit's items of this tile begin: totals of the lower digits, counts of the tiles before
    {
        const int a = totals[2 * tid], b = totals[2 * tid + 1];
        const int inc = wave_scan(a + b, lane);
        if (lane == 63) sm[wave] = inc;
        __syncthreads();
        int e = inc - a - b;
        for (int w = 0; w < wave; ++w) e += sm[w];
        base[2 * tid] = e + counts[(long long)(2 * tid) * tiles + blockIdx.x];
        base[2 * tid + 1] = e + a + counts[(long long)(2 * tid + 1) * tiles + blockIdx.x];
    }
    const int first = blockIdx.x * LTILE + wave * (LROUNDS * 64) + lane;
    unsigned key[LROUNDS];
    int rank[LROUNDS];
    for (int r = 0; r < LROUNDS; ++r) {
        const int i = first + r * 64;
        key[r] = i < in.n ? sort_key(in, i) : ~0u;
    }
    __syncthreads();
    for (int r = 0; r < LROUNDS; ++r) {
        const unsigned d = (key[r] >> shift) & (LBINS - 1);
        int total;
        const int low = lower_peers<LB>(d, lane, &total);
        const int before = cnt[wave][d];
        __builtin_amdgcn_wave_barrier();
        rank[r] = before + low;
        if (low == total - 1) cnt[wave][d] = (unsigned short)(before + total);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for (int d = tid; d < LBINS; d += 256) {
        int s = 0;
        for (int w = 0; w < LWAVES; ++w) {
            const int c = cnt[w][d];
            cnt[w][d] = (unsigned short)s;
            s += c;
        }
    }
    __syncthreads();
    for (int r = 0; r < LROUNDS; ++r) {
        const int i = first + r * 64;
        if (i < in.n) {                                          // (the items behind the last rank behind all others: no gap)
            const unsigned d = (key[r] >> shift) & (LBINS - 1);
            const int to = base[d] + cnt[wave][d] + rank[r];
            keys_out[to] = key[r];
            pos_out[to] = in.ids ? i : in.pos[i];
            if (touched && key[r] < (unsigned)in.n_entries) touched[key[r]] = 1;
        }
    }
}

// ---- sums ------------------------------------------------------------------------------------------------------------------
constexpr int UNROLL = 8;               // rows in flight per wavefront: 8 KB, 128 KB on a compute unit with 16 wavefronts

template <typename T, bool ALIGNED>
__device__ __forceinline__ int column(int chunk, int lane, int j) {
    constexpr int V = Vec<T>::N;
    return chunk * 64 * V + (ALIGNED ? lane * V + j : j * 64 + lane);
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void load_cols(const T* row, int chunk, int lane, int dim, float* v) {
    constexpr int V = Vec<T>::N;
    if constexpr (ALIGNED) {
        const int c = column<T, true>(chunk, lane, 0);
        if (c < dim) Vec<T>::load(row + c, v);
    } else {
        for (int j = 0; j < V; ++j) {
            const int c = column<T, false>(chunk, lane, j);
            v[j] = c < dim ? (float)row[c] : 0.f;
        }
    }
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void write_row(T* row, int chunk, int lane, int dim, const float* acc, float scale, int accumulate) {
    constexpr int V = Vec<T>::N;
    float v[V];
    if (accumulate) load_cols<T, ALIGNED>(row, chunk, lane, dim, v);
    for (int j = 0; j < V; ++j) v[j] = accumulate ? v[j] + scale * acc[j] : scale * acc[j];
    if constexpr (ALIGNED) {
        const int c = column<T, true>(chunk, lane, 0);
        if (c < dim) Vec<T>::store(row + c, v);
    } else {
        for (int j = 0; j < V; ++j) {
            const int c = column<T, false>(chunk, lane, j);
            if (c < dim) row[c] = (T)v[j];
        }
    }
}

// pieces of the runs that cross a border: [tile][0: began before the tile, 1: goes on behind it][chunk][j][lane]
template <int V>
__device__ __forceinline__ float* piece(float* pieces, int tile, int which, int chunk, int chunks) {
    return pieces + (((long long)tile * 2 + which) * chunks + chunk) * (64 * V);
}

template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256) void sum_k(const unsigned* __restrict__ keys, const int* __restrict__ pos, int n,
                                             const T* __restrict__ dy, long long ldy, int dim, long long n_entries, float scale,
                                             T* __restrict__ dtable, int accumulate, int tile_len, int tiles, int chunks,
                                             float* __restrict__ pieces, const unsigned char* __restrict__ touched, int sum_blocks) {
    constexpr int V = Vec<T>::N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int)blockIdx.x >= sum_blocks) {                          // rows without an id
        const float zero[V] = {};
        const long long step = (long long)(gridDim.x - sum_blocks) * 4;
        for (long long v = (long long)(blockIdx.x - sum_blocks) * 4 + wave; v < n_entries; v += step)
            if (!touched[v])
                for (int c = 0; c < chunks; ++c) write_row<T, ALIGNED>(dtable + v * dim, c, lane, dim, zero, 0.f, 0);
        return;
    }
    const long long item = (long long)blockIdx.x * 4 + wave;
    const int tile = (int)(item / chunks), chunk = (int)(item - (long long)tile * chunks);
    if (tile >= tiles) return;
    const int t0 = tile * tile_len, all = min(tile_len, n - t0);
    const unsigned key_l = lane < all ? keys[t0 + lane] : ~0u;
    const int pos_l = lane < all ? pos[t0 + lane] : 0;
    const int cnt = __popcll(__ballot(key_l < (unsigned)n_entries));      // sorted: what is not summed is behind the rest
    if (cnt == 0) return;
    unsigned cur = (unsigned)__builtin_amdgcn_readlane((int)key_l, 0);
    bool head = t0 > 0 && keys[t0 - 1] == cur;
    float acc[V];
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    auto leave = [&](int which) {
        float* q = piece<V>(pieces, tile, which, chunk, chunks);
        for (int j = 0; j < V; ++j) q[j * 64 + lane] = acc[j];
    };
    for (int j0 = 0; j0 < cnt; j0 += UNROLL) {
        float v[UNROLL][V];
        unsigned k[UNROLL];
        for (int u = 0; u < UNROLL; ++u) {
            const int i = min(j0 + u, cnt - 1);
            k[u] = j0 + u < cnt ? (unsigned)__builtin_amdgcn_readlane((int)key_l, i) : ~0u;
            const int p = __builtin_amdgcn_readlane(pos_l, i);
            load_cols<T, ALIGNED>(dy + (long long)p * ldy, chunk, lane, dim, v[u]);
        }
        for (int u = 0; u < UNROLL; ++u) {
            if (j0 + u >= cnt) break;
            if (k[u] != cur) {
                if (head) leave(0);
                else write_row<T, ALIGNED>(dtable + (long long)cur * dim, chunk, lane, dim, acc, scale, accumulate);
                cur = k[u];
                head = false;
                for (int j = 0; j < V; ++j) acc[j] = 0.f;
            }
            for (int j = 0; j < V; ++j) acc[j] += v[u][j];
        }
    }
    if (head) leave(0);
    else if (t0 + cnt < n && keys[t0 + cnt] == cur) leave(1);
    else write_row<T, ALIGNED>(dtable + (long long)cur * dim, chunk, lane, dim, acc, scale, accumulate);
}

// A workgroup per (tile, chunk) that a crossing run begins in: eight wavefronts add every eighth piece, then each other's sums.
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(512) void join_k(const unsigned* __restrict__ keys, int n, int dim, long long n_entries, float scale,
                                              T* __restrict__ dtable, int accumulate, int tile_len, int chunks,
                                              float* __restrict__ pieces) {
    constexpr int V = Vec<T>::N;
    __shared__ float sm[8][64 * V];
    const int tile = blockIdx.x / chunks, chunk = blockIdx.x - tile * chunks;
    const int t0 = tile * tile_len, t1 = t0 + tile_len;
    if (t1 >= n) return;
    const unsigned cur = keys[t1 - 1];
    if (cur >= (unsigned)n_entries || keys[t1] != cur) return;
    if (t0 > 0 && keys[t0 - 1] == cur) return;                    // began in an earlier tile
    int lo = t1, hi = n;                                          // first position behind the run
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (keys[mid] == cur) lo = mid + 1;
        else hi = mid;
    }
    const int last = (lo - 1) / tile_len;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float acc[V];
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    for (int t = tile + wave; t <= last; t += 8) {
        const float* q = piece<V>(pieces, t, t == tile ? 1 : 0, chunk, chunks);
        for (int j = 0; j < V; ++j) acc[j] += q[j * 64 + lane];
    }
    for (int j = 0; j < V; ++j) sm[wave][j * 64 + lane] = acc[j];
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < 8; ++w)
            for (int j = 0; j < V; ++j) acc[j] += sm[w][j * 64 + lane];
        write_row<T, ALIGNED>(dtable + (long long)cur * dim, chunk, lane, dim, acc, scale, accumulate);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
int tile_len_of(long long n) { return n <= SMALL ? 16 : 64; }     // few positions: more wavefronts

struct Layout {
    long long keys[2], pos[2], counts, totals, pieces, touched, bytes;
};
Layout layout(long long n, int dim, long long n_entries) {
    Layout l;
    long long at = 0;
    auto take = [&](long long b) {
        const long long here = at;
        at += round_up(b, 256);
        return here;
    };
    const bool small = n <= SMALL;
    const long long tiles = cdiv(n, LTILE), cols = round_up(dim, 512);
    for (int k = 0; k < 2; ++k) {
        l.keys[k] = k && small ? l.keys[0] : take(4 * n);
        l.pos[k] = k && small ? l.pos[0] : take(4 * n);
    }
    l.counts = take(small ? 0 : 4 * LBINS * tiles);
    l.totals = take(4 * LBINS);
    l.pieces = take(4 * 2 * cols * cdiv(n, tile_len_of(n)));
    l.touched = take(n_entries);
    l.bytes = at;
    return l;
}

bool valid_sizes(long long n, int dim, long long n_entries) {
    return n >= 0 && n < (1LL << 31) - 65536 && dim > 0 && dim <= (1 << 24) && n_entries > 0 && n_entries < (1LL << 30);
}

template <typename T, bool ALIGNED>
int launch_sums(const unsigned* keys, const int* pos, int n, const void* dy, long long ldy, int dim, long long n_entries, float scale,
                void* dtable, int accumulate, float* pieces, const unsigned char* touched, hipStream_t st) {
    const int tl = tile_len_of(n), tiles = cdiv(n, tl), chunks = cdiv(dim, 64 * Vec<T>::N);
    const long long blocks = ((long long)tiles * chunks + 3) / 4;
    if (blocks + 4096 > 0x7fffffffLL) return S2AG_E_UNSUPPORTED;
    long long zero = 0;
    if (touched) zero = n_entries / 4 + 1 < 4096 ? n_entries / 4 + 1 : 4096;
    if (blocks + zero)
        hipLaunchKernelGGL((sum_k<T, ALIGNED>), dim3((unsigned)(blocks + zero)), dim3(256), 0, st, keys, pos, n,
                           static_cast<const T*>(dy), ldy, dim, n_entries, scale, static_cast<T*>(dtable), accumulate, tl, tiles,
                           chunks, pieces, touched, (int)blocks);
    S2AG_LAUNCH_CHECK();
    if (tiles > 1) {
        hipLaunchKernelGGL((join_k<T, ALIGNED>), dim3((unsigned)((long long)(tiles - 1) * chunks)), dim3(512), 0, st, keys, n, dim, n_entries,
                           scale, static_cast<T*>(dtable), accumulate, tl, chunks, pieces);
        S2AG_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T>
int launch_lookup(const void* ids, int ids_i32, const void* table, long long n, int dim, long long n_entries, float scale, void* out,
                  hipStream_t st) {
    constexpr int V = Vec<T>::N;
    const bool al = dim % V == 0 && aligned16(table) && aligned16(out);
    const int per_row = al ? dim / V : dim;
    int tx = 0;
    while (tx < 8 && (1 << tx) < per_row) ++tx;
    const long long rows = 256 >> tx;
    long long blocks = (n + rows - 1) / rows;
    if (blocks > 8192) blocks = 8192;
    if (al)
        hipLaunchKernelGGL((lookup_k<T, true>), dim3((unsigned)blocks), dim3(256), 0, st, ids, ids_i32, static_cast<const T*>(table), n, dim,
                           n_entries, scale, static_cast<T*>(out), tx);
    else
        hipLaunchKernelGGL((lookup_k<T, false>), dim3((unsigned)blocks), dim3(256), 0, st, ids, ids_i32, static_cast<const T*>(table), n, dim,
                           n_entries, scale, static_cast<T*>(out), tx);
    S2AG_LAUNCH_CHECK();
    return 0;
}
}  // namespace

extern "C" int s2ag_emb_lookup(const void* ids, int ids_i32, const void* table, int bf16, long long n, int dim, long long n_entries,
                               float scale, void* out, void* stream) {
    if (!valid_sizes(n, dim, n_entries) || !table || (n && (!ids || !out))) return S2AG_E_BADARG;
    if (n == 0) return 0;
    return bf16 ? launch_lookup<bf16_t>(ids, ids_i32, table, n, dim, n_entries, scale, out, (hipStream_t)stream)
                : launch_lookup<float>(ids, ids_i32, table, n, dim, n_entries, scale, out, (hipStream_t)stream);
}

extern "C" long long s2ag_emb_grad_workspace_bytes(long long n, int dim, long long n_entries) {
    if (!valid_sizes(n, dim, n_entries)) return S2AG_E_BADARG;
    return layout(n, dim, n_entries).bytes;
}

extern "C" int s2ag_emb_grad(const void* ids, int ids_i32, const void* dy, long long ldy, int bf16, long long n, int dim,
                             long long n_entries, long long padding_idx, float scale, void* dtable, int accumulate, void* workspace,
                             long long workspace_bytes, void* stream) {
    if (!valid_sizes(n, dim, n_entries) || !dtable || (n && (!ids || !dy || !workspace || ldy < dim)) || (accumulate && bf16))
        return S2AG_E_BADARG;
    const Layout l = layout(n, dim, n_entries);
    if (!workspace || workspace_bytes < l.bytes || !aligned16(workspace)) return S2AG_E_BADARG;
    hipStream_t st = (hipStream_t)stream;
    char* ws = static_cast<char*>(workspace);
    unsigned char* touched = accumulate ? nullptr : reinterpret_cast<unsigned char*>(ws + l.touched);
    unsigned* keys = reinterpret_cast<unsigned*>(ws + l.keys[0]);
    int* pos = reinterpret_cast<int*>(ws + l.pos[0]);
    int bits = 1;
    while ((n_entries >> bits) != 0) ++bits;                       // the keys 0 .. n_entries
    const bool small = n <= SMALL;
    const bool clear_inside = small && n > 0 && n_entries <= 131072;
    if (touched && !clear_inside)
        if (hipError_t e = zero_async(touched, (size_t)round_up(n_entries, 4), st)) return (int)e;
    if (n > 0 && small) {
        hipLaunchKernelGGL(sort_small_k, dim3(1), dim3(1024), 0, st, ids, ids_i32, (int)n, n_entries, padding_idx, cdiv(bits, SB),
                           (int)clear_inside, keys, pos, touched);
        S2AG_LAUNCH_CHECK();
    } else if (n > 0) {
        const int tiles = cdiv(n, LTILE), passes = cdiv(bits, LB);
        int* counts = reinterpret_cast<int*>(ws + l.counts);
        int* totals = reinterpret_cast<int*>(ws + l.totals);
        SortIn in{ids, ids_i32, n_entries, padding_idx, nullptr, nullptr, (int)n};
        for (int p = 0; p < passes; ++p) {
            const int to = (passes - 1 - p) & 1;                   // the last pass ends in the first pair of buffers
            unsigned* ko = reinterpret_cast<unsigned*>(ws + l.keys[to]);
            int* po = reinterpret_cast<int*>(ws + l.pos[to]);
            hipLaunchKernelGGL(sort_count_k, dim3(tiles), dim3(256), 0, st, in, p * LB, tiles, counts);
            S2AG_LAUNCH_CHECK();
            hipLaunchKernelGGL(sort_scan_k, dim3(LBINS), dim3(256), 0, st, tiles, counts, totals);
            S2AG_LAUNCH_CHECK();
            hipLaunchKernelGGL(sort_move_k, dim3(tiles), dim3(256), 0, st, in, p * LB, tiles, counts, totals, ko, po,
                               p == passes - 1 ? touched : nullptr);
            S2AG_LAUNCH_CHECK();
            in.ids = nullptr;
            in.keys = ko;
            in.pos = po;
        }
    }
    float* pieces = reinterpret_cast<float*>(ws + l.pieces);
    const int V = bf16 ? 8 : 4;
    const bool al = dim % V == 0 && ldy % V == 0 && aligned16(dy) && aligned16(dtable);
#define S2AG_SUMS(T, AL) launch_sums<T, AL>(keys, pos, (int)n, dy, ldy, dim, n_entries, scale, dtable, accumulate, pieces, touched, st)
    if (bf16) return al ? S2AG_SUMS(bf16_t, true) : S2AG_SUMS(bf16_t, false);
    return al ? S2AG_SUMS(float, true) : S2AG_SUMS(float, false);
#undef S2AG_SUMS
}
