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
// Measured, 65536 ids of a table of 131072 x 2048, bf16: lookup 81 us (268 MB read, 268 written: 6.6 TB/s); gradient 211 us, of them
// sorting 31, sums and zeros 172 (268 MB read, 537 written: 4.7 TB/s), joins 8.  4352 ids of a table of 20000 x 300, fp32: 5 us
// and 34.  A copy of 2 GB runs at 4.7 TB/s.
//
// ids that are not in the table, and the padding row's, sort behind the last row under the key n_entries and are not summed.
#include "text_common.h"

namespace {
using namespace s2ag;
using namespace s2ag::text;

// ---- lookup ----------------------------------------------------------------------------------------------------------------
// A row is read by 2^tx_log lanes, 16 bytes each, four rows in flight: with one, a workgroup waits for an id and then for a row
// for every 4 KB that it writes.
template <typename T>
__global__ __launch_bounds__(256) void lookup_k(const void* __restrict__ ids, int ids_i32, const T* __restrict__ table, long long n,
                                                int dim, long long n_entries, float scale, T* __restrict__ out, int tx_log) {
    constexpr int V = Vec<T>::N, R = 4;
    const int tx = threadIdx.x & ((1 << tx_log) - 1), ty = threadIdx.x >> tx_log, rows = 256 >> tx_log;
    for (long long r0 = (long long)blockIdx.x * rows * R + ty; r0 < n; r0 += (long long)gridDim.x * rows * R) {
        const T* src[R];
        bool in[R];
        for (int u = 0; u < R; ++u) {
            const long long r = r0 + u * rows, id = r < n ? load_id(ids, ids_i32, r) : -1;
            in[u] = id >= 0 && id < n_entries;
            src[u] = table + (in[u] ? id : 0) * dim;
        }
        for (int c = tx * V; c < dim; c += V << tx_log) {
            if (c + V <= dim) {
                float v[R][V];
                for (int u = 0; u < R; ++u) Vec<T>::load_any(src[u] + c, v[u]);
                for (int u = 0; u < R; ++u) {
                    for (int j = 0; j < V; ++j) v[u][j] = in[u] ? v[u][j] * scale : 0.f;
                    if (r0 + u * rows < n) Vec<T>::store_any(out + (r0 + u * rows) * dim + c, v[u]);
                }
            } else {
                for (int u = 0; u < R; ++u)
                    for (int j = c; j < dim; ++j)
                        if (r0 + u * rows < n) out[(r0 + u * rows) * dim + j] = in[u] ? (T)((float)src[u][j] * scale) : (T)0.f;
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

// Up to SMALL positions: one workgroup sorts them in LDS in one launch, 8 bits a pass (4352 positions: 13 us; the four launches that
// more positions take 23; 8192: 19 and 25).  Items go by wavefront, round and lane, which is their
// order; a wavefront counts its items per digit while it ranks them, so that a pass reads its items once.
constexpr int SMALL = 8192;
constexpr int SB = 8, SBINS = 1 << SB, SWAVES = 16;
template <int SROUNDS>
__global__ __launch_bounds__(1024) void sort_small_k(const void* __restrict__ ids, int ids_i32, int n, long long n_entries,
                                                     long long padding_idx, int passes, int clear_flags,
                                                     unsigned* __restrict__ keys, int* __restrict__ pos,
                                                     unsigned char* __restrict__ touched) {
    __shared__ unsigned k_s[SROUNDS * 1024];
    __shared__ unsigned short p_s[SROUNDS * 1024];
    __shared__ unsigned short cnt[SWAVES][SBINS];
    __shared__ int base[SBINS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (touched && clear_flags)
        for (long long i = tid; i < (n_entries + 15) / 16; i += 1024) reinterpret_cast<u32x4*>(touched)[i] = u32x4{0, 0, 0, 0};      // (padded)
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

// More: per pass of LB bits one launch counts the digits of every tile of LTILE items and one moves the items.  Up to DIRECT
// tiles the second adds the counts of the tiles itself; more are added up by a launch between the two (a workgroup per digit).
// (32 tiles: 32 us in four launches, 32 in six; 64 tiles: 34 and 32; 128 tiles: 46 and 40)
constexpr int LB = 9, LBINS = 1 << LB, LTILE = 2048, LWAVES = 4, LROUNDS = LTILE / 256, DIRECT = 32;
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
// counts: [tile][digit] for the direct sums, [digit][tile] for the launch between
__device__ __forceinline__ long long count_at(int tile, int digit, int tiles) {
    return tiles <= DIRECT ? (long long)tile * LBINS + digit : (long long)digit * tiles + tile;
}

__global__ __launch_bounds__(256) void sort_count_k(SortIn in, int shift, int tiles, int* __restrict__ counts,
                                                    unsigned char* __restrict__ clear) {
    __shared__ int c[LBINS];
    if (clear)                                                   // the flags that the last pass sets (padded to 16)
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (in.n_entries + 15) / 16; i += (long long)gridDim.x * 256)
            reinterpret_cast<u32x4*>(clear)[i] = u32x4{0, 0, 0, 0};
    for (int i = threadIdx.x; i < LBINS; i += 256) c[i] = 0;
    __syncthreads();
    const int t0 = blockIdx.x * LTILE;
    unsigned key[LROUNDS];
    for (int r = 0; r < LROUNDS; ++r) {
        const int i = t0 + r * 256 + threadIdx.x;
        key[r] = i < in.n ? sort_key(in, i) : 0u;
    }
    for (int r = 0; r < LROUNDS; ++r)
        if (t0 + r * 256 + (int)threadIdx.x < in.n) atomicAdd(&c[(key[r] >> shift) & (LBINS - 1)], 1);     // (whole numbers: any order, one sum)
    __syncthreads();
    for (int i = threadIdx.x; i < LBINS; i += 256) counts[count_at(blockIdx.x, i, tiles)] = c[i];
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
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, me = blockIdx.x;
    const int first = me * LTILE + wave * (LROUNDS * 64) + lane;
    unsigned key[LROUNDS];
    int at[LROUNDS], rank[LROUNDS];
    for (int r = 0; r < LROUNDS; ++r) {
        const int i = first + r * 64;
        key[r] = i < in.n ? sort_key(in, i) : ~0u;
        at[r] = in.ids || i >= in.n ? i : in.pos[i];
    }
    for (int i = tid; i < LWAVES * LBINS; i += 256) (&cnt[0][0])[i] = 0;
    // where each digit's items of this tile begin: totals of the lower digits, counts of the tiles before
    {
        int total[2] = {0, 0}, before[2] = {0, 0};
        if (tiles <= DIRECT) {
#pragma unroll 8
            for (int t = 0; t < tiles; ++t)
                for (int h = 0; h < 2; ++h) {
                    const int c = counts[(long long)t * LBINS + 2 * tid + h];
                    total[h] += c;
                    if (t < me) before[h] += c;
                }
        } else {
            for (int h = 0; h < 2; ++h) {
                total[h] = totals[2 * tid + h];
                before[h] = counts[count_at(me, 2 * tid + h, tiles)];
            }
        }
        const int inc = wave_scan(total[0] + total[1], lane);
        if (lane == 63) sm[wave] = inc;
        __syncthreads();
        int e = inc - total[0] - total[1];
        for (int w = 0; w < wave; ++w) e += sm[w];
        base[2 * tid] = e + before[0];
        base[2 * tid + 1] = e + total[0] + before[1];
    }
    for (int r = 0; r < LROUNDS; ++r) {                          // (a wavefront's counters are its own)
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
        if (first + r * 64 < in.n) {                             // (the items behind the last rank behind all others: no gap)
            const unsigned d = (key[r] >> shift) & (LBINS - 1);
            const int to = base[d] + cnt[wave][d] + rank[r];
            keys_out[to] = key[r];
            pos_out[to] = at[r];
            if (touched && key[r] < (unsigned)in.n_entries) touched[key[r]] = 1;
        }
    }
}

// ---- sums ------------------------------------------------------------------------------------------------------------------
constexpr int ZERO_ROWS = 64;           // a lane to each: 16 of them take as long
constexpr int UNROLL = 8;               // rows in flight per wavefront: 8 KB, 128 KB on a compute unit with 16 wavefronts

// A lane's V columns of a row: one 16-byte access at any alignment, element by element at the row's end.
template <typename T>
__device__ __forceinline__ void load_cols(const T* row, int c, int dim, float* v) {
    constexpr int V = Vec<T>::N;
    if (c + V <= dim) {
        Vec<T>::load_any(row + c, v);
    } else {
        for (int j = 0; j < V; ++j) v[j] = c + j < dim ? (float)row[c + j] : 0.f;
    }
}

template <typename T>
__device__ __forceinline__ void write_cols(T* row, int c, int dim, const float* acc, float scale, int accumulate) {
    constexpr int V = Vec<T>::N;
    float v[V];
    if (accumulate) load_cols<T>(row, c, dim, v);
    for (int j = 0; j < V; ++j) v[j] = accumulate ? v[j] + scale * acc[j] : scale * acc[j];
    if (c + V <= dim) {
        Vec<T>::store_any(row + c, v);
    } else {
        for (int j = 0; j < V; ++j)
            if (c + j < dim) row[c + j] = (T)v[j];
    }
}

// A wavefront writes zeros to n elements: rows that follow each other are one piece of memory.
template <typename T>
__device__ __forceinline__ void write_zeros(T* p, long long n, int lane) {
    constexpr int V = Vec<T>::N;
    const long long head = min((long long)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)), n), body = (n - head) / V;
    if (lane < head) p[lane] = (T)0.f;
    u32x4* q = reinterpret_cast<u32x4*>(p + head);
    for (long long i = lane; i < body; i += 64) q[i] = u32x4{0, 0, 0, 0};
    if (lane < n - head - body * V) p[head + body * V + lane] = (T)0.f;
}

// pieces of the runs that cross a border: [tile][0: began before the tile, 1: goes on behind it][chunk][j][lane]
template <int V>
__device__ __forceinline__ float* piece(float* pieces, int tile, int which, int chunk, int chunks) {
    return pieces + (((long long)tile * 2 + which) * chunks + chunk) * (64 * V);
}

template <typename T>
__global__ __launch_bounds__(256) void sum_k(const unsigned* __restrict__ keys, const int* __restrict__ pos, int n,
                                             const T* __restrict__ dy, long long ldy, int dim, long long n_entries, float scale,
                                             T* __restrict__ dtable, int accumulate, int tile_len, int tiles, int chunks,
                                             float* __restrict__ pieces, const unsigned char* __restrict__ touched, int sum_blocks) {
    constexpr int V = Vec<T>::N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int)blockIdx.x >= sum_blocks) {                          // rows without an id, ZERO_ROWS to a wavefront
        const long long v0 = ((long long)(blockIdx.x - sum_blocks) * 4 + wave) * ZERO_ROWS;
        const bool mine = v0 + lane < n_entries && !touched[v0 + lane];
        unsigned long long left = __ballot(mine);
        while (left) {
            const int at = __ffsll(left) - 1;
            const unsigned long long rest = ~(left >> at);
            const int run = rest ? __ffsll(rest) - 1 : 64;
            write_zeros<T>(dtable + (v0 + at) * dim, (long long)run * dim, lane);
            left = at + run >= 64 ? 0 : left & ~(((1ULL << run) - 1) << at);
        }
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
    const int c = (chunk * 64 + lane) * V;
    float acc[V];
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    auto leave = [&](int which) {
        float* q = piece<V>(pieces, tile, which, chunk, chunks);
        for (int j = 0; j < V; ++j) q[j * 64 + lane] = acc[j];
    };
    for (int j0 = 0; j0 < cnt; j0 += UNROLL) {
        float v[UNROLL][V];
        unsigned k[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int i = min(j0 + u, cnt - 1);
            k[u] = (unsigned)__builtin_amdgcn_readlane((int)key_l, i);
            const int p = __builtin_amdgcn_readlane(pos_l, i);
            load_cols<T>(dy + (long long)p * ldy, c, dim, v[u]);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            if (j0 + u < cnt) {
                if (k[u] != cur) {
                    if (head) leave(0);
                    else write_cols<T>(dtable + (long long)cur * dim, c, dim, acc, scale, accumulate);
                    cur = k[u];
                    head = false;
                    for (int j = 0; j < V; ++j) acc[j] = 0.f;
                }
                for (int j = 0; j < V; ++j) acc[j] += v[u][j];
            }
        }
    }
    if (head) leave(0);
    else if (t0 + cnt < n && keys[t0 + cnt] == cur) leave(1);
    else write_cols<T>(dtable + (long long)cur * dim, c, dim, acc, scale, accumulate);
}

// Runs that cross a border, a wavefront to the (tile, chunk) that one begins in.  Most end in the next tile: the wavefront adds
// their pieces by itself.  Of a long one its workgroup's eight wavefronts add every eighth piece, then each other's sums.  (5 us for
// 65536 positions of 2048 columns; 89 us where half of a million positions of 64 columns hold one id, whose 7800 pieces are one
// workgroup's.)
constexpr int JOINERS = 8;
template <typename T>
__global__ __launch_bounds__(64 * JOINERS) void join_k(const unsigned* __restrict__ keys, int n, int dim, long long n_entries,
                                                       float scale, T* __restrict__ dtable, int accumulate, int tile_len, int tiles,
                                                       int chunks, float* __restrict__ pieces) {
    constexpr int V = Vec<T>::N;
    __shared__ float sm[JOINERS][64 * V];
    __shared__ int last_s[JOINERS];
    __shared__ unsigned cur_s[JOINERS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tile0 = (int)(blockIdx.x / chunks) * JOINERS, tile = tile0 + wave, chunk = blockIdx.x % chunks;
    auto add = [&](float* acc, int tile, int from, int last, int step) {
#pragma unroll 8
        for (int t = from; t <= last; t += step) {
            const float* q = piece<V>(pieces, t, t == tile ? 1 : 0, chunk, chunks);
            for (int j = 0; j < V; ++j) acc[j] += q[j * 64 + lane];
        }
    };
    int last = -1;
    unsigned cur = ~0u;
    if (tile < tiles - 1) {                                       // (the last tile has no border behind it)
        const int t0 = tile * tile_len, t1 = t0 + tile_len;
        cur = keys[t1 - 1];
        if (cur < (unsigned)n_entries && keys[t1] == cur && !(t0 > 0 && keys[t0 - 1] == cur)) {
            // the first tile whose last key is another one, or the last tile: 64 tiles looked at, then by halves
            const int t = min(tile + 1 + lane, tiles - 1);
            const unsigned long long other = __ballot(t == tiles - 1 || keys[(t + 1) * tile_len - 1] != cur);
            if (other) {
                last = min(tile + __ffsll(other), tiles - 1);
            } else {
                int lo = tile + 65, hi = tiles - 1;
                while (lo < hi) {
                    const int mid = lo + ((hi - lo) >> 1);
                    if (keys[(mid + 1) * tile_len - 1] == cur) lo = mid + 1;
                    else hi = mid;
                }
                last = lo;
            }
            if (keys[last * tile_len] != cur) --last;            // (the run ends with the tile before)
        }
    }
    const bool alone = last >= 0 && last - tile < 2 * JOINERS;
    if (alone) {
        float acc[V];
        for (int j = 0; j < V; ++j) acc[j] = 0.f;
        add(acc, tile, tile, last, 1);
        write_cols<T>(dtable + (long long)cur * dim, (chunk * 64 + lane) * V, dim, acc, scale, accumulate);
    }
    if (lane == 0) {
        last_s[wave] = alone ? -1 : last;
        cur_s[wave] = cur;
    }
    __syncthreads();
    for (int w = 0; w < JOINERS; ++w) {
        if (last_s[w] < 0) continue;                              // (the same for the whole workgroup)
        float acc[V];
        for (int j = 0; j < V; ++j) acc[j] = 0.f;
        add(acc, tile0 + w, tile0 + w + wave, last_s[w], JOINERS);
        for (int j = 0; j < V; ++j) sm[wave][j * 64 + lane] = acc[j];
        __syncthreads();
        if (wave == 0) {
            for (int o = 1; o < JOINERS; ++o)
                for (int j = 0; j < V; ++j) acc[j] += sm[o][j * 64 + lane];
            write_cols<T>(dtable + (long long)cur_s[w] * dim, (chunk * 64 + lane) * V, dim, acc, scale, accumulate);
        }
        __syncthreads();
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// Short tiles where long ones are fewer than sixteen wavefronts for each of 256 compute units (sums and joins, bf16, 512 columns:
// 65536 positions 72 us with 64, 42 with 16; 131072 66 and 58; 262144 97 and 117)
int tile_len_of(long long n, int chunks) { return cdiv(n, 64) * (long long)chunks < 4096 ? 16 : 64; }

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
    l.pieces = take(4 * 2 * cols * cdiv(n, tile_len_of(n, cdiv(dim, 512))));      // (bf16 has the fewer chunks)
    l.touched = take(n_entries);        // (a multiple of 256: cleared in 16-byte steps)
    l.bytes = at;
    return l;
}

bool valid_sizes(long long n, int dim, long long n_entries) {
    return n >= 0 && n < (1LL << 31) - 65536 && dim > 0 && dim <= (1 << 24) && n_entries > 0 && n_entries < (1LL << 30);
}

template <typename T>
int launch_sums(const unsigned* keys, const int* pos, int n, const void* dy, long long ldy, int dim, long long n_entries, float scale,
                void* dtable, int accumulate, float* pieces, const unsigned char* touched, hipStream_t st) {
    const int chunks = cdiv(dim, 64 * Vec<T>::N), tl = tile_len_of(n, chunks), tiles = cdiv(n, tl);
    const long long blocks = ((long long)tiles * chunks + 3) / 4;
    const long long zero = touched ? (n_entries + 4 * ZERO_ROWS - 1) / (4 * ZERO_ROWS) : 0;
    if (blocks + zero > 0x7fffffffLL || (long long)tiles * chunks > 0x7fffffffLL) return S2AG_E_UNSUPPORTED;
    if (blocks + zero)
        hipLaunchKernelGGL(sum_k<T>, dim3((unsigned)(blocks + zero)), dim3(256), 0, st, keys, pos, n, static_cast<const T*>(dy), ldy, dim,
                           n_entries, scale, static_cast<T*>(dtable), accumulate, tl, tiles, chunks, pieces, touched, (int)blocks);
    S2AG_LAUNCH_CHECK();
    if (tiles > 1) {
        hipLaunchKernelGGL(join_k<T>, dim3((unsigned)(cdiv(tiles - 1, JOINERS) * (long long)chunks)), dim3(64 * JOINERS), 0, st, keys,
                           n, dim, n_entries, scale, static_cast<T*>(dtable), accumulate, tl, tiles, chunks, pieces);
        S2AG_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T>
int launch_lookup(const void* ids, int ids_i32, const void* table, long long n, int dim, long long n_entries, float scale, void* out,
                  hipStream_t st) {
    const int per_row = cdiv(dim, Vec<T>::N);
    int tx = 0;
    while (tx < 8 && (1 << tx) < per_row) ++tx;
    const long long rows = 4 * (256 >> tx);
    long long blocks = (n + rows - 1) / rows;
    if (blocks > (1 << 20)) blocks = 1 << 20;
    hipLaunchKernelGGL(lookup_k<T>, dim3((unsigned)blocks), dim3(256), 0, st, ids, ids_i32, static_cast<const T*>(table), n, dim, n_entries,
                       scale, static_cast<T*>(out), tx);
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
    const bool clear_inside = n > 0 && (!small || n_entries <= 131072);        // by the sort's first launch (0.7 us of its one workgroup for 131072 rows; a launch of its own 2.4)
    if (touched && !clear_inside)
        if (hipError_t e = zero_async(touched, (size_t)round_up(n_entries, 4), st)) return (int)e;
    if (n > 0 && small) {
#define S2AG_SORT(R) \
    hipLaunchKernelGGL(sort_small_k<R>, dim3(1), dim3(1024), 0, st, ids, ids_i32, (int)n, n_entries, padding_idx, cdiv(bits, SB), \
                       (int)clear_inside, keys, pos, touched)
        if (n <= 1024) S2AG_SORT(1);
        else if (n <= 2048) S2AG_SORT(2);
        else if (n <= 4096) S2AG_SORT(4);
        else if (n <= 6144) S2AG_SORT(6);
        else S2AG_SORT(8);
#undef S2AG_SORT
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
            hipLaunchKernelGGL(sort_count_k, dim3(tiles), dim3(256), 0, st, in, p * LB, tiles, counts, p == 0 ? touched : nullptr);
            S2AG_LAUNCH_CHECK();
            if (tiles > DIRECT) {
                hipLaunchKernelGGL(sort_scan_k, dim3(LBINS), dim3(256), 0, st, tiles, counts, totals);
                S2AG_LAUNCH_CHECK();
            }
            hipLaunchKernelGGL(sort_move_k, dim3(tiles), dim3(256), 0, st, in, p * LB, tiles, counts, totals, ko, po,
                               p == passes - 1 ? touched : nullptr);
            S2AG_LAUNCH_CHECK();
            in.ids = nullptr;
            in.keys = ko;
            in.pos = po;
        }
    }
    float* pieces = reinterpret_cast<float*>(ws + l.pieces);
    return bf16 ? launch_sums<bf16_t>(keys, pos, (int)n, dy, ldy, dim, n_entries, scale, dtable, accumulate, pieces, touched, st)
                : launch_sums<float>(keys, pos, (int)n, dy, ldy, dim, n_entries, scale, dtable, accumulate, pieces, touched, st);
}
