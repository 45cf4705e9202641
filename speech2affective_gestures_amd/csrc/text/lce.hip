// Softmax cross entropy of a linear layer over a large vocabulary, without keeping the logits, and its gradient.
//
//   z = X W^T        loss_i = log sum_v exp z_iv - z_{i,t_i}
//   G = g_i (softmax(z)_iv - [v = t_i])        dX = G W        dW = G^T X
//
// Bound by the matrix pipe: 2 N V D operations for the loss, 8 N V D with the gradient (the logits are formed twice: keeping
// them would be N V values, the largest tensor of a training step by far).
//
// All four products are ONE tiled product out[r][c] = sum_k R[r][k] Q[c][k] on bf16 matrix instructions with four ends: (1) max
// and sum of exponentials of each row of a tile of logits, joined over the tiles by a small launch; (2) G of a piece of the
// vocabulary, stored; (3) dX += G W over that piece in fp32; (4) dW of that piece.  Where k runs down the columns of an operand
// as it lies in memory (W in (3), G and X in (4)) its fragments come by the transposing LDS read: nothing is transposed in memory.
//
// The rows that are ignored are left out of every product: the others are packed in front (rowmap), their number stays on the
// device, and the tiles behind it end at once.
//
// fp32 operands are taken in pieces on the same instructions, at more than the rate of the f32 ones.  For the logits as two
// halves of 11 bits each (a power of two to every row, so that its largest value is near the top of the type's range): three
// products; the fourth is 2^-22 of the whole, as is what the halves leave (2^-39 of the row's largest value where that is more,
// for values below 2^-17 of it).  Six products of bf16 pieces took 32 us for the logits of 136 rows and 20 000 words of 300
// values, these take 22.  For the gradient's products as three bf16 pieces (v = p0 + p1 + p2 to 2^-25) and the six products that
// matter at fp32's own rounding: G has values of many magnitudes in a row, which bf16's range holds and a half's does not.
// bf16 operands need one product; there G is rounded to bf16 (2^-8 of each value at most; sums stay in fp32), without its factor g where
// that is one number for all rows.
//
// Measured, 7373 of 8192 rows counting, 131072 words of 2048 values, bf16: max and sum 3.0 ms (1320 TFLOP/s), G 3.3 (1190), dX 3.1
// (1290), dW 2.9 (1360); a library product of 8192 cubed ran at 1280, of 16384 cubed at 1540.  136 rows, 20000 words of 300 values,
// fp32: 22, 29, 30 and 28 us, packing 24, the joins and sums 16: there nothing fills the card, and launches and the ends of tiles
// are most of it.
#include "text_common.h"
#include <algorithm>
#include <type_traits>

namespace {
using namespace s2ag;
using namespace s2ag::text;

typedef _Float16 f16_t;
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

constexpr int BK = 64;                  // k of a stage: 128-byte rows in LDS, eight 16-byte slots
constexpr int ROWS = 256;               // packed rows are padded to this

struct State {                          // what the forward call leaves for the backward call
    int* count;
    int *rowmap, *inv, *tgt;            // packed -> row, row -> packed or -1, packed targets (-1: not in the vocabulary)
    float* lse;
};
long long padded(long long rows) { return round_up(rows, ROWS); }
long long state_words(long long rows) { return 64 + 2 * round_up(rows, 64) + 2 * padded(rows); }
State state_of(void* p, long long rows) {
    int* w = static_cast<int*>(p);
    State s;
    s.count = w;
    s.rowmap = w + 64;
    s.inv = s.rowmap + round_up(rows, 64);
    s.tgt = s.inv + round_up(rows, 64);
    s.lse = reinterpret_cast<float*>(s.tgt + padded(rows));
    return s;
}

// ---- rows that have a target, packed in order --------------------------------------------------------------------------------
struct Select {
    const void* target;
    int i32;
    long long rows, vocab, ignore;
    State s;
    float* loss_rows;
};
__device__ __forceinline__ void select_rows(const Select& q) {   // one workgroup of 1024
    const long long rows = q.rows, vocab = q.vocab, ignore = q.ignore;
    const State& s = q.s;
    __shared__ int sm[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int base = 0;
    for (long long r0 = 0; r0 < rows; r0 += 1024) {
        const long long r = r0 + threadIdx.x;
        const long long t = r < rows ? load_id(q.target, q.i32, r) : ignore;
        const bool keep = t != ignore;
        const unsigned long long m = __ballot(keep);
        if (lane == 0) sm[wave] = __popcll(m);
        __syncthreads();
        int at = base + __popcll(m & ((1ULL << lane) - 1));
        for (int w = 0; w < 16; ++w) {
            if (w < wave) at += sm[w];
            base += sm[w];
        }
        if (keep) {
            s.rowmap[at] = (int)r;
            s.tgt[at] = t >= 0 && t < vocab ? (int)t : -1;
        }
        if (r < rows) {
            s.inv[r] = keep ? at : -1;
            if (q.loss_rows && !keep) q.loss_rows[r] = 0.f;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) *s.count = base;
}
__global__ __launch_bounds__(1024) void select_rows_k(Select q) { select_rows(q); }

// ---- operands: rows of features, padded with zeros to a multiple of 64, fp32 as three bf16 pieces --------------------------------
struct Operand {
    const bf16_t* p;
    long long plane, ld;                // elements
};

__device__ __forceinline__ void split3(float v, bf16_t* q) {
    const float most = 3.3895313892515355e38f;                   // bf16's largest: fp32's own would round to an infinity
    q[0] = fabsf(v) < INFINITY ? (bf16_t)fminf(fmaxf(v, -most), most) : (bf16_t)v;
    const float r1 = v - (float)q[0];   // exact
    q[1] = (bf16_t)r1;
    q[2] = (bf16_t)(r1 - (float)q[1]);
}

// Rows of the packed operand that are written: all of W, or the live rows of X and zeros up to a multiple of 256.
__device__ __forceinline__ long long packed_rows(const int* count, long long rows, long long* live) {
    *live = count ? (long long)*count : rows;
    return count ? (*live + ROWS - 1) / ROWS * ROWS : rows;
}
template <typename T>
__device__ __forceinline__ void load8(const T* s, int c, int dim, bool in, float* v) {
    if (in && c + 8 <= dim) {
        for (int j = 0; j < 8; j += Vec<T>::N) Vec<T>::load_any(s + c + j, v + j);
    } else {
        for (int j = 0; j < 8; ++j) v[j] = in && c + j < dim ? (float)s[c + j] : 0.f;
    }
}

// What a packing launch does: rows of `src` by way of rowmap, or all of them, to `dst` or to the halves, powers and pieces.
template <typename T> struct Pack;
template <> struct Pack<bf16_t> {
    const bf16_t* src;
    long long ld;
    int dim, kp;
    const int *rowmap, *count;
    long long rows;
    bf16_t* dst;
};
template <> struct Pack<float> {
    const float* src;
    long long ld;
    int dim, kp;
    const int *rowmap, *count;
    long long rows;
    f16_t* halves;
    int* power;
    bf16_t* pieces;                     // may be null
    long long plane;
};

// dst[r][0..kp) from row rowmap[r] (or r) of src, zeros behind column dim
__device__ __forceinline__ void pack_rows(const Pack<bf16_t>& q, unsigned block, unsigned blocks) {
    const bf16_t* __restrict__ src = q.src;
    bf16_t* __restrict__ dst = q.dst;
    const int* rowmap = q.rowmap;
    const long long ld = q.ld;
    const int dim = q.dim, kp = q.kp, groups = kp / 8;
    long long live;
    const long long end = packed_rows(q.count, q.rows, &live);
    const long long total = end * groups;
    for (long long i = (long long)block * blockDim.x + threadIdx.x; i < total; i += (long long)blocks * blockDim.x) {
        const long long r = i / groups;
        const int c = (int)(i - r * groups) * 8;
        const bool in = r < live;
        float v[8];
        load8(src + (in ? (rowmap ? (long long)rowmap[r] : r) : 0) * ld, c, dim, in, v);
        Vec<bf16_t>::store(dst + r * kp + c, v);
    }
}

// The same of fp32, a wavefront to a row: two halves, the row times 2^-power[r] of them, and three bf16 pieces if they are wanted.
// An infinity leaves NaN in the pieces behind it, as its products would anyway.
__device__ __forceinline__ void pack_rows(const Pack<float>& p, unsigned block, unsigned blocks) {
    const float* __restrict__ src = p.src;
    f16_t* __restrict__ halves = p.halves;
    bf16_t* __restrict__ pieces = p.pieces;
    int* __restrict__ power = p.power;
    const int* rowmap = p.rowmap;
    const long long ld = p.ld, plane = p.plane;
    const int dim = p.dim, kp = p.kp, waves = blockDim.x >> 6;
    long long live;
    const long long end = packed_rows(p.count, p.rows, &live);
    const int lane = threadIdx.x & 63;
    for (long long r = (long long)block * waves + (threadIdx.x >> 6); r < end; r += (long long)blocks * waves) {
        const bool in = r < live;
        const float* s = src + (in ? (rowmap ? (long long)rowmap[r] : r) : 0) * ld;
        float top = 0.f;
        for (int c = lane * 8; c < kp; c += 512) {
            float v[8];
            load8(s, c, dim, in, v);
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
        }
        for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
        int up = 0;
        if (top > 0.f && top < INFINITY) {
            frexpf(top, &up);
            up = 15 - up;                                        // the largest value to 2^14 .. 2^15
        }
        if (lane == 0) power[r] = -up;
        for (int c = lane * 8; c < kp; c += 512) {
            float v[8];
            load8(s, c, dim, in, v);
            f16x8 h[2];
            bf16x8 q[3];
            for (int j = 0; j < 8; ++j) {
                const float t = ldexpf(v[j], up);
                h[0][j] = (f16_t)t;
                h[1][j] = (f16_t)(t - (float)h[0][j]);           // (the difference is exact)
                bf16_t piece[3];
                split3(v[j], piece);
                for (int k = 0; k < 3; ++k) q[k][j] = piece[k];
            }
            for (int k = 0; k < 2; ++k) *reinterpret_cast<f16x8*>(halves + k * plane + r * kp + c) = h[k];
            if (pieces)
                for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8*>(pieces + k * plane + r * kp + c) = q[k];
        }
    }
}

template <typename T> __global__ __launch_bounds__(256) void pack_k(Pack<T> q) { pack_rows(q, blockIdx.x, gridDim.x); }
// W does not wait for the rows: its packing and their selection are one launch.
template <typename T> __global__ __launch_bounds__(1024) void select_and_pack_k(Select s, Pack<T> q) {
    if (blockIdx.x == 0) select_rows(s);
    else pack_rows(q, blockIdx.x - 1, gridDim.x - 1);
}

// ---- the tiled product -------------------------------------------------------------------------------------------------------
enum End { STATS, GRADS, ACCUM, STORE };

struct Product {
    Operand r, q;
    long long r_rows, q_rows;           // rows of out, columns of out that exist; what lies behind reads as zeros
    // an operand whose k runs down its columns: its rows (k) and columns that exist
    long long r_deep, q_deep;
    int r_cols, q_cols;
    int k;                              // of one pair of pieces, a multiple of 64
    const int* k_count;                 // not null: k is this, rounded up to 64
    const int* r_count;                 // not null: rows of R that matter
    bool fp32;                          // operands in pieces
    // STATS, GRADS of fp32: rows of R and Q times 2^power are what is multiplied
    const int *r_power, *q_power;
    int tiles_q;
    int splits, slots;                  // the most parts of k; workgroups that run at a time
    // STATS: max and sum of exponentials [tile_q][padded rows], logit of the target
    const int* tgt;
    long long q0;                       // word number of Q's first row
    long long vocab;
    float2* part;
    long long part_ld;
    float* target_logit;
    // GRADS: [row][word] pitch g_ld; the factor of each row is grad_out[rowmap[row]], if it is not one for all
    const float *lse, *grad_out;
    const int* rowmap;
    bf16_t* g;
    long long g_ld, g_plane;
    // ACCUM: fp32 [split][row, padded to the tile][col] pitch out_ld; STORE: rows of dW
    void* out;
    long long out_ld;
    int cols, add, out_bf16;
    const float* scale;                 // STORE: not null: the factor of all rows, over their number with `mean`
    int mean;
};

// Pairs of pieces, two bits each, every one with a piece of R or Q from the one before it, which is then not requested again (7
// requests of 12, or 4 of 6): (0, 2) (0, 1) (1, 1) (1, 0) (0, 0) (2, 0) of three pieces, (0, 1) (0, 0) (1, 0) of two.  One bit to a
// pair: R, or Q, is another piece than before.
template <int PAIRS> struct Pairs {
    static constexpr int r = PAIRS == 6 ? 0x850 : 0x10, q = PAIRS == 6 ? 0x016 : 0x01, r_new = PAIRS == 6 ? 0x35 : 0x5, q_new = PAIRS == 6 ? 0x0b : 0x3;
};

typedef short s16x4_t __attribute__((ext_vector_type(4)));
#define S2AG_LDS_PTR(type, p) ((__attribute__((address_space(3))) type*)(p))

// 16-byte slot of (row, slot) in a stage: the slots of a row are permuted by the row's low bits, so that the 16 rows that a
// wavefront reads at one slot lie in different banks.
__device__ __forceinline__ int slot_at(int row, int slot) { return row * BK + ((slot ^ (row & 7)) << 3); }

// A raw buffer descriptor: base address, no stride, bytes behind which a lane reads zeros.
__device__ __forceinline__ u32x4 buffer(const void* p, unsigned bytes) {
    const unsigned long long a = reinterpret_cast<unsigned long long>(p);
    return u32x4{(unsigned)a, (unsigned)(a >> 32), bytes, 0x00020000u};
}

typedef __attribute__((address_space(3))) bf16_t* LdsPtr;       // (from a general pointer the compiler tests for null every time)

// 16 bytes a lane from the buffer to LDS: lane l's land at dst + 16 l.
__device__ __forceinline__ void to_lds(u32x4 from, LdsPtr dst, unsigned lane_offset, int offset) {
    __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(from[0] | (unsigned long long)from[1] << 32), 0, (int)from[2], (int)from[3]);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, lane_offset, offset, 0, 0);
}
// The same, written out: behind the builtin the compiler lets every transposing read wait for all requests that are out.  No
// register is loaded, and the waits for LDS are the kernel's own.  (Only where there are such reads: it costs 2 to 8 %.)
__device__ __forceinline__ void to_lds_beside_transposing_reads(u32x4 from, LdsPtr dst, unsigned lane_offset, int offset) {
    const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)dst);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(at), "v"(lane_offset), "s"(from), "s"(offset) : "memory");
}

// Matrix instruction with its accumulator in the accumulation registers, where the compiler, left to itself, moves a set that
// fills all 256 of them to and fro.  The compiler knows no matrix instruction here: `settle` stands between the last of them
// and the first use of a result, and between the zeros and the first of them.
__device__ __forceinline__ void mfma_acc(f32x4& c, bf16x8 a, bf16x8 b) {
    asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_acc_halves(f32x4& c, bf16x8 a, bf16x8 b) {
    asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// One of its values, read where it is used (the compiler would read all 256 at once and not find registers for them).
__device__ __forceinline__ float acc_read(float a) {
    float v;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(a));
    return v;
}
// A barrier for LDS alone: stores to memory stay out (__syncthreads would wait for them).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // (keeps what follows behind the barrier)
}
__device__ __forceinline__ void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// exp(d): two terms of the argument's product with log2 e for fp32 operands, one for bf16 ones, whose logits carry more than that
template <bool PRECISE>
__device__ __forceinline__ float exp_of(float d) {
    if constexpr (!PRECISE) return __expf(d);
    d = d < -150.f ? -150.f : d;                                 // (0 in fp32 either way; an infinity has no rest)
    const float t = d * 1.44269504088896340736f;
    const float rest = fmaf(d, 1.44269504088896340736f, -t) + d * 1.925963033500935e-8f;     // log2 e - its fp32 value
    const float e = exp2f(t);
    return fmaf(e * 0.693147180559945f, rest, e);
}

// The factor of all rows.  Where none counts there is nothing that it enters: an infinite one leaves the zeros as they are.
__device__ __forceinline__ float scale_of(const float* scale, int mean, int kept) {
    if (kept == 0) return 1.f;
    return mean ? *scale / (float)kept : *scale;
}

constexpr int GROUP = 8;                // row tiles that the columns pass by at a time

// The tiles of a launch, in the order in which they are handed out; everything here is one for the workgroup.
struct Tiles {
    int n, splits, per, tiles_r, kt;
    int stages, more;                   // of a part of k; so many parts have one more
};
__host__ __device__ inline int splits_of(int tiles, int most, int slots) {       // few tiles: k is split to fill the card
    const int s = tiles > 0 ? slots / tiles : 1;
    return s < 1 ? 1 : s > most ? most : s;
}

// f(0), f(STEP), ... below N, with the index as a constant: the accumulators are registers, which no loop can index.
template <int I, int N, int STEP, typename F>
__device__ __forceinline__ void each(F f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        each<I + STEP, N, STEP>(f);
    }
}

// A tile of values to out[row][column], rows below `live` and columns below p.cols.
template <typename T, int BR, int BQ, int WR, int WQ, typename F>
__device__ __forceinline__ void write_out(bf16_t* scratch, T* out, const Product& p, long long r0, long long c0, int live, float f, F value) {
    constexpr int NT = 64 * WR * WQ, TR = BR / WR, TQ = BQ / WQ, RI = TR / 16, QI = TQ / 16;
    constexpr int V = Vec<T>::N, SLOTS = BQ / V, JS = 4 / (int)sizeof(T);         // 32 or 16 rows of each part at a time
    T* const lds = reinterpret_cast<T*>(scratch);
    auto at = [](int row, int slot) { return row * BQ + ((slot ^ (row & 15)) * V); };
    const int lane = threadIdx.x & 63, fl = lane & 15, fk = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wave / WQ, wq = wave % WQ;
    const bool vectors = (p.out_ld % V == 0) && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    each<0, RI, JS>([&](auto at_j) {
        constexpr int jj = decltype(at_j)::value;
#pragma unroll
        for (int j = jj; j < jj + JS; ++j) {
#pragma unroll
            for (int i = 0; i < QI; ++i) {
                const int lrow = wr * 16 * JS + (j - jj) * 16 + fl, col = wq * TQ + i * 16 + fk * 4;
                T* o = lds + at(lrow, col / V) + col % V;
                if constexpr (sizeof(T) == 2) {
                    bf16x4 q;
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[e] = (bf16_t)(value(i, j, e) * f);
                    *reinterpret_cast<bf16x4*>(o) = q;
                } else {
                    f32x4 q;
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[e] = value(i, j, e) * f;
                    *reinterpret_cast<f32x4*>(o) = q;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        lds_barrier();
        for (int i = threadIdx.x; i < WR * 16 * JS * SLOTS; i += NT) {
            const int lrow = i / SLOTS, slot = i % SLOTS;
            const long long row = r0 + lrow / (16 * JS) * TR + jj * 16 + lrow % (16 * JS), c = c0 + slot * V;
            if (row >= live || c >= p.cols) continue;
            float v[V];
            Vec<T>::load(lds + at(lrow, slot), v);
            T* o = out + row * p.out_ld + c;
            if (vectors && c + V <= p.cols) {
                if (sizeof(T) == 4 && p.add) {
                    float w[V];
                    Vec<T>::load(o, w);
                    for (int e = 0; e < V; ++e) v[e] += w[e];
                }
                Vec<T>::store(o, v);
            } else {
                for (int e = 0; e < V; ++e)
                    if (c + e < p.cols) o[e] = (T)(p.add ? (float)o[e] + v[e] : v[e]);
            }
        }
        lds_barrier();
    });
}

// An operand's tile in LDS.  k along its rows: [row][64 k], slots of 16 bytes permuted by slot_at.  k down its columns: [k][B
// columns], pairs of slots (the 16 columns of a fragment) permuted by four bits of k, so that the 16 rows that a transposing read
// touches lie in different banks.
template <int B>
__device__ __forceinline__ int pair_at(int k, int pair) { return k * B + ((pair ^ (((k & 3) | ((k >> 3) & 3) << 2) & (B / 16 - 1))) << 4); }

// byte offset in the operand of the 16 bytes that a thread brings with request i
template <int B, bool DOWN, int NT>
__device__ __forceinline__ unsigned request_at(int i, int tid, long long ld) {
    const int at = i * NT + tid;                                 // 16-byte place in the tile
    if constexpr (DOWN) {
        const int k = at / (B / 8), slot = at % (B / 8);
        return (unsigned)(k * ld * 2 + (pair_at<B>(k, slot >> 1) - k * B + (slot & 1) * 8) * 2);
    } else {
        const int row = at >> 3;
        return (unsigned)(row * ld * 2 + ((at & 7) ^ (row & 7)) * 16);
    }
}

// Where a lane finds its part of the operand's fragments (16 rows or columns each) from x on.  k along the rows: place n is that of
// half n of a stage, the fragments 16 rows apart; down the columns: place n is that of fragment n, the halves 32 rows apart.
template <int B, bool DOWN>
__device__ __forceinline__ LdsPtr fragment_place(LdsPtr tile, int x, int n, int fl, int fk) {
    if constexpr (!DOWN) return tile + slot_at(x + fl, n * 4 + fk);
    else return tile + pair_at<B>(fk * 8 + (fl >> 2), (x >> 4) + n) + (fl & 3) * 4;
}
// k = 32 ks + 8 fk + 0..7 of the fragment
template <int B, bool DOWN>
__device__ __forceinline__ bf16x8 fragment(LdsPtr at) {
    if constexpr (!DOWN) {
        return *(__attribute__((address_space(3))) const bf16x8*)at;
    } else {
        bf16x8 v;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bf16x4 y = __builtin_bit_cast(
                bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(at + h * 4 * B)));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[h * 4 + e] = y[e];
        }
        return v;
    }
}

template <int BR, int BQ, int WR, int WQ, End END, bool PRECISE>
__global__ __launch_bounds__(64 * WR * WQ, BR == 256 ? 1 : 2) void product_k(Product p) {
    constexpr int NT = 64 * WR * WQ;
    constexpr int TR = BR / WR, TQ = BQ / WQ, RI = TR / 16, QI = TQ / 16;      // a wavefront's part
    constexpr int LR = BR * 8 / NT, LQ = BQ * 8 / NT;                          // 16-byte loads per thread and stage
    constexpr int STAGE = (BR + BQ) * BK;
    constexpr bool RK = END == STORE, QK = END == STORE || END == ACCUM;       // k runs down the operand's columns
    extern __shared__ __attribute__((aligned(16))) bf16_t lds[];
    const LdsPtr r_tiles = (LdsPtr)lds, q_tiles = r_tiles + 2 * BR * BK;       // two of each
    bf16_t* const scratch = lds + 2 * STAGE;                                   // 64 x BQ, for the ends
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave / WQ, wq = wave % WQ;
    constexpr bool HALVES = PRECISE && (END == STATS || END == GRADS);
    constexpr int pairs = HALVES ? 3 : PRECISE ? 6 : 1;
    // (read here: a load that is still out behind the end of a tile would be waited for in every stage of the next one)
    float f = 1.f;
    if constexpr (END == STORE) {
        if (p.scale) f = scale_of(p.scale, p.mean, *p.k_count);
        f = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(f)));
    }

    // (whole-number division runs on the vector units: the results are told to be one for the wavefront, so that the operands'
    // descriptors stay in scalar registers)
    const int live = p.r_count ? __builtin_amdgcn_readfirstlane(*p.r_count) : (int)p.r_rows;
    Tiles ts;
    ts.tiles_r = __builtin_amdgcn_readfirstlane((live + BR - 1) / BR);
    ts.splits = __builtin_amdgcn_readfirstlane(splits_of(ts.tiles_r * p.tiles_q, p.splits, p.slots));
    ts.kt = p.k_count ? __builtin_amdgcn_readfirstlane((*p.k_count + BK - 1) / BK) : p.k / BK;
    ts.stages = __builtin_amdgcn_readfirstlane(ts.kt * pairs / ts.splits);
    ts.more = ts.kt * pairs - ts.stages * ts.splits;
    ts.per = GROUP * p.tiles_q;
    ts.n = ts.tiles_r * p.tiles_q * ts.splits;

    // A workgroup takes many tiles, so that the operands of the next one are on their way while this one ends.  Workgroups are
    // dealt to the eight XCDs in turn; each XCD gets a contiguous range of tiles, and inside it the tiles go column by column
    // over GROUP row tiles, so that the tiles that run at the same time share operands in its L2.  (8192 rows,
    // 131072 words of 2048 values: 12.3 ms with groups of 8 or 4, 12.7 of 2.)
    const int xcd = blockIdx.x & 7, step = gridDim.x >> 3;
    const int last = __builtin_amdgcn_readfirstlane((int)((long long)ts.n * (xcd + 1) / 8));
    const int first = __builtin_amdgcn_readfirstlane((int)((long long)ts.n * xcd / 8)) + (blockIdx.x >> 3);
    if (first >= last) return;

    struct Place {
        long long r0, c0;
        int split, it0, it1;
    };
    auto place = [&](int v) {
        Place t;
        t.split = __builtin_amdgcn_readfirstlane(v / (ts.tiles_r * p.tiles_q));
        v -= t.split * ts.tiles_r * p.tiles_q;
        const int grp = __builtin_amdgcn_readfirstlane(v / ts.per), g0 = grp * GROUP, gsz = min(ts.tiles_r - g0, GROUP);
        t.r0 = (long long)__builtin_amdgcn_readfirstlane(g0 + (v - grp * ts.per) % gsz) * BR;
        t.c0 = (long long)__builtin_amdgcn_readfirstlane((v - grp * ts.per) / gsz) * BQ;
        t.it0 = ts.stages * t.split + min(t.split, ts.more);
        t.it1 = t.it0 + ts.stages + (t.split < ts.more ? 1 : 0);
        return t;
    };

    unsigned r_off[LR], q_off[LQ];
#pragma unroll
    for (int i = 0; i < LR; ++i) r_off[i] = request_at<BR, RK, NT>(i, tid, p.r.ld);
#pragma unroll
    for (int i = 0; i < LQ; ++i) q_off[i] = request_at<BQ, QK, NT>(i, tid, p.q.ld);

    // the stage that is requested next: its tile, pair of pieces and place along k; behind the last one the descriptors are
    // empty, so that the loop has no branch
    constexpr bool REUSE = pairs > 1;
    int next = first - step, pair = 0, kk = 0, left = 0;
    int r_new = 1, q_new = 1, r_to_buf = 1, q_to_buf = 1, r_last = 1, q_last = 1;          // (REUSE)
    long long r0_next = 0, c0_next = 0;
    u32x4 rr, qr, r_base, q_base;
    // an operand's part of that stage: from row x of R or Q, or from its column x on
    auto descriptor = [&](const Operand& o, bool down, long long x, long long rows, int tile, long long deep, int cols) {
        const bf16_t* at = o.p;
        long long bytes;
        if (down) {
            const long long k0 = (long long)kk * BK, n = deep - k0 < BK ? deep - k0 : BK;
            at += k0 * o.ld + x;
            bytes = n > 0 ? ((n - 1) * o.ld + cols - x) * 2 : 0;
        } else {
            const long long n = rows - x < tile ? rows - x : tile;
            at += x * o.ld;
            bytes = n > 0 ? n * o.ld * 2 : 0;                    // (a tile may lie behind the words)
        }
        return buffer(at, left > 0 ? (unsigned)bytes : 0u);
    };
    int whole = 0;                                               // stages from here on that no end of a column cuts
    const unsigned long long r_step = 2ULL * BK * p.r.ld, q_step = 2ULL * BK * p.q.ld;
    auto descriptors = [&]() {
        rr = descriptor(p.r, RK, r0_next, p.r_rows, BR, p.r_deep, p.r_cols);
        qr = descriptor(p.q, QK, c0_next, p.q_rows, BQ, p.q_deep, p.q_cols);
        if (QK) whole = (int)((RK && p.r_deep < p.q_deep ? p.r_deep : p.q_deep) / BK) - kk;
    };
    auto move = [](u32x4& d, unsigned long long bytes) {
        const unsigned long long at = (d[0] | (unsigned long long)d[1] << 32) + bytes;
        d[0] = (unsigned)at;
        d[1] = (unsigned)(at >> 32);
    };
    // Of the pair's pieces what is in LDS stays there: its requests get an empty descriptor, so that there are always as many of
    // them to wait for, and put zeros where nothing lies that is still read.
    auto aim = [&](bool all) {
        r_new = all ? 1 : (Pairs<pairs>::r_new >> pair) & 1;
        q_new = all ? 1 : (Pairs<pairs>::q_new >> pair) & 1;
        rr = r_base;
        qr = q_base;
        move(rr, 2ULL * p.r.plane * ((Pairs<pairs>::r >> (2 * pair)) & 3));
        move(qr, 2ULL * p.q.plane * ((Pairs<pairs>::q >> (2 * pair)) & 3));
        if (!r_new) rr[2] = 0;
        if (!q_new) qr[2] = 0;
        r_to_buf = r_last ^ 1;
        q_to_buf = q_last ^ 1;
        r_last ^= r_new;
        q_last ^= q_new;
    };
    auto next_tile = [&]() {
        left = 0;
        for (next += step; next < last; next += step) {
            const Place t = place(next);
            left = t.it1 - t.it0;
            if (left <= 0) continue;                             // (no stage: nothing to request)
            kk = REUSE ? __builtin_amdgcn_readfirstlane(t.it0 / pairs) : t.it0;
            pair = t.it0 - kk * pairs;
            r0_next = t.r0;
            c0_next = t.c0;
            break;
        }
        descriptors();
        if constexpr (REUSE) {
            r_base = rr;
            q_base = qr;
            aim(true);
        }
    };
    auto next_k = [&]() {
        ++kk;
        if (QK) {                                                // down the columns: few scalar instructions, the matrix unit waits for them
            if constexpr (REUSE) {
                rr = r_base;
                qr = q_base;
            }
            if (--whole > 0) {
                if (RK) move(rr, r_step);
                move(qr, q_step);
            } else {
                descriptors();
            }
            if constexpr (REUSE) {
                r_base = rr;
                q_base = qr;
            }
        }
    };
    auto advance = [&]() {
        if (--left <= 0) {
            next_tile();
        } else if constexpr (REUSE) {
            if (++pair == pairs) {
                pair = 0;
                next_k();
            }
            aim(false);
        } else {
            next_k();
        }
    };
    // requests [from, from + n) of the LR + LQ of a stage
    auto issue = [&](int buf, int from, int n) {
        const LdsPtr r_to = r_tiles + (REUSE ? r_to_buf : buf) * (BR * BK) + wave * 512;
        const LdsPtr q_to = q_tiles + (REUSE ? q_to_buf : buf) * (BQ * BK) + wave * 512;
        const int off = kk * (BK * 2);                           // (down the columns the descriptor moves)
#pragma unroll
        for (int i = from; i < from + n; ++i) {
            const u32x4 from = i < LR ? rr : qr;
            const LdsPtr to = i < LR ? r_to + i * NT * 8 : q_to + (i - LR) * NT * 8;
            const unsigned lane_offset = i < LR ? r_off[i < LR ? i : 0] : q_off[i < LR ? 0 : i - LR];
            const int move = (i < LR ? RK : QK) ? 0 : off;
            if constexpr (QK) to_lds_beside_transposing_reads(from, to, lane_offset, move);
            else to_lds(from, to, lane_offset, move);
        }
    };

    f32x4 acc[QI][RI];
    const int fl = lane & 15, fk = lane >> 4;
    // The places in the stage that is read; on to the other one of the two and back.  (As few vector instructions as can be: the
    // matrix unit waits for them too.)
    constexpr int RN = RK ? RI : 2, QN = QK ? QI : 2;
    LdsPtr r_place[RN], q_place[QN];
#pragma unroll
    for (int n = 0; n < RN; ++n) r_place[n] = fragment_place<BR, RK>(r_tiles, wr * TR, n, fl, fk);
#pragma unroll
    for (int n = 0; n < QN; ++n) q_place[n] = fragment_place<BQ, QK>(q_tiles, wq * TQ, n, fl, fk);
    int r_other = BR * BK, q_other = BQ * BK, r_go = 0, q_go = 0;
    auto read_q = [&](bf16x8 (&a)[QI], int ks, int i) {
        if constexpr (QK) a[i] = fragment<BQ, QK>(q_place[i] + ks * 32 * BQ);
        else a[i] = fragment<BQ, QK>(q_place[ks] + i * 16 * BK);
    };
    auto read_r = [&](bf16x8 (&b)[RI], int ks, int j) {
        if constexpr (RK) b[j] = fragment<BR, RK>(r_place[j] + ks * 32 * BR);
        else b[j] = fragment<BR, RK>(r_place[ks] + j * 16 * BK);
    };
    auto multiply = [&](const bf16x8& a, const bf16x8& b, int i, int j) {
        if constexpr (RI * QI * 4 == 256 && HALVES) mfma_acc_halves(acc[i][j], a, b);
        else if constexpr (RI * QI * 4 == 256) mfma_acc(acc[i][j], a, b);
        else if constexpr (HALVES) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc[i][j], 0, 0, 0);
        else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc[i][j], 0, 0, 0);
    };
    auto value = [&](int i, int j, int e) {
        if constexpr (RI * QI * 4 == 256) return acc_read(acc[i][j][e]);
        else return acc[i][j][e];
    };

    // Two stages in LDS, two halves of a stage in registers.  While the first half of a stage is multiplied its second half is
    // read, R before Q: when every wavefront has its part of R, R's place is free and the R of the stage after the next is
    // requested; in the middle of the stage all of it is read, the next stage (requested a stage ago) has landed, and while the
    // second half is multiplied the first half of the next stage is read and the Q of the stage after it is requested.
    // A wavefront is alone on its matrix unit, which waits for whatever stands between two of its instructions for longer than
    // one of them takes.  So reads and requests are dealt out singly: a fragment behind every PER-th matrix instruction of the
    // first half of the groups (the others cover the reads' way), a request behind every RPER-th or QPER-th.
    constexpr int G = QI, M = QI * RI, EARLY = (G / 2 - 1) * RI, PER = M / 2 / (QI + RI), RPER = (M - EARLY - 1) / LR, QPER = M / LQ;
    static_assert(M / 2 % (QI + RI) == 0 && M % LQ == 0 && RI * PER <= EARLY, "dealing out");
    auto deal = [&](bf16x8 (&a)[QI], bf16x8 (&b)[RI], int ks, int m) {       // what follows matrix instruction m
        if (m < M / 2 && m % PER == 0) {
            const int u = m / PER;
            if (ks == 0) {                                       // (the first reads of the other stage)
                if (RK ? u < RI : u == 0)
                    for (int n = RK ? u : 0; n < (RK ? u + 1 : RN); ++n) r_place[n] += REUSE ? r_go : r_other;
                if (QK ? u >= RI : u == RI)
                    for (int n = QK ? u - RI : 0; n < (QK ? u - RI + 1 : QN); ++n) q_place[n] += REUSE ? q_go : q_other;
            }
            if (u < RI) read_r(b, ks, u);
            else read_q(a, ks, u - RI);
        }
    };
    bf16x8 a0[QI], b0[RI], a1[QI], b1[RI];
#pragma unroll 1
    for (int b = 0; b < 2; ++b) {
        advance();
        issue(b, 0, LR + LQ);
        if (b) break;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < RI; ++j) read_r(b0, 0, j);
#pragma unroll
    for (int i = 0; i < QI; ++i) read_q(a0, 0, i);
    int buf = 0;
    for (int tile = first; tile < last; tile += step) {
        const Place t = place(tile);
#pragma unroll
        for (int i = 0; i < QI; ++i)
#pragma unroll
            for (int j = 0; j < RI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        settle();
        for (int n = t.it0; n < t.it1; ++n) {
            if constexpr (REUSE) {                               // to the next stage's pieces, if they are others
                r_go = r_new ? r_other : 0;
                q_go = q_new ? q_other : 0;
            }
            each<0, M, 1>([&](auto at_m) {
                constexpr int m = decltype(at_m)::value;
                if constexpr (m == (M > 16 ? EARLY : 0)) advance();          // (scalar work, where little or nothing waits for it)
                if constexpr (m == EARLY) {
                    // (the reads of Q that were dealt out behind R's are still out)
                    constexpr int OUT = (EARLY / PER - RI) * (QK ? 2 : 1);
                    static_assert(OUT == 0 || OUT == 4 || OUT == 8, "");
                    if constexpr (OUT == 8) asm volatile("s_waitcnt lgkmcnt(8)" ::: "memory");
                    else if constexpr (OUT == 4) asm volatile("s_waitcnt lgkmcnt(4)" ::: "memory");
                    else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("s_waitcnt lgkmcnt(15)" ::: "memory");      // (keeps the requests behind the barrier)
                }
                multiply(a0[m / RI], b0[m % RI], m / RI, m % RI);
                __builtin_amdgcn_sched_barrier(0);
                deal(a1, b1, 1, m);
                if (m > EARLY && (m - EARLY) % RPER == 0 && (m - EARLY) / RPER <= LR) issue(buf, (m - EARLY) / RPER - 1, 1);
                __builtin_amdgcn_sched_barrier(0);
            });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if constexpr (LR == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
            static_assert(LR == 8 || LR == 4, "the requests for R of the stage after the next stay out");
            __builtin_amdgcn_s_barrier();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (keeps the reads behind the barrier)
            each<0, M, 1>([&](auto at_m) {
                constexpr int m = decltype(at_m)::value;
                multiply(a1[m / RI], b1[m % RI], m / RI, m % RI);
                __builtin_amdgcn_sched_barrier(0);
                deal(a0, b0, 0, m);
                if (m % QPER == QPER - 1) issue(buf, LR + m / QPER, 1);
                __builtin_amdgcn_sched_barrier(0);
            });
            buf ^= 1;
            if constexpr (REUSE) {
                r_other = r_go ? -r_other : r_other;
                q_other = q_go ? -q_other : q_other;
            } else {
                r_other = -r_other;
                q_other = -q_other;
            }
        }
        settle();

        // element e of acc[i][j]: column i * 16 + fk * 4 + e, row j * 16 + fl of the wavefront's part
        const long long wr0 = t.r0 + wr * TR, wc0 = t.c0 + wq * TQ;
        if constexpr (END == STATS || END == GRADS) {
            const int word0 = (int)(p.q0 + wc0) + fk * 4;        // the lane's first word
            const int words = (int)p.vocab - word0;              // that it may use, counted from there
            const bool edge = p.q0 + t.c0 + BQ > p.vocab;
            // logits of fp32: the rows' and words' powers of two come back, the words' by way of LDS (behind what the ends use)
            int* const word_power = reinterpret_cast<int*>(scratch + 32 * BQ);
            int row_power[RI];
            if constexpr (HALVES) {
                for (int i = tid; i < BQ; i += NT) word_power[i] = p.q_power[t.c0 + i];
#pragma unroll
                for (int j = 0; j < RI; ++j) row_power[j] = p.r_power[wr0 + j * 16 + fl];
                lds_barrier();
            }
            auto logits = [&](int j, float (&z)[QI * 4]) {
#pragma unroll
                for (int i = 0; i < QI; ++i) {
                    int4 w;
                    if constexpr (HALVES) w = *reinterpret_cast<const int4*>(word_power + wq * TQ + i * 16 + fk * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        z[i * 4 + e] = value(i, j, e);
                        if constexpr (HALVES) z[i * 4 + e] = ldexpf(z[i * 4 + e], row_power[j] + (e == 0 ? w.x : e == 1 ? w.y : e == 2 ? w.z : w.w));
                    }
                }
            };
            if constexpr (END == STATS) {
                float2* sm = reinterpret_cast<float2*>(scratch);     // [WQ][BR]
                int tgt[RI];
#pragma unroll
                for (int j = 0; j < RI; ++j) tgt[j] = wr0 + j * 16 + fl < live ? p.tgt[wr0 + j * 16 + fl] : -1;
#pragma unroll
                for (int j = 0; j < RI; ++j) {
                    const int row = (int)wr0 + j * 16 + fl;
                    const unsigned at = (unsigned)(tgt[j] - word0);  // the target's place, if it is the lane's
                    float z[QI * 4], m4[4], s4[4] = {0.f, 0.f, 0.f, 0.f};
                    logits(j, z);
                    if (edge) {
#pragma unroll
                        for (int i = 0; i < QI * 4; ++i)
                            if (i / 4 * 16 + i % 4 >= words) z[i] = -INFINITY;
                    }
                    if (at < (unsigned)TQ && (at & 12) == 0) {       // (four columns of sixteen are the lane's)
                        float logit = z[0];
#pragma unroll
                        for (int i = 1; i < QI * 4; ++i) logit = at == (unsigned)(i / 4 * 16 + i % 4) ? z[i] : logit;
                        p.target_logit[row] = logit;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) m4[e] = z[e];
#pragma unroll
                    for (int i = 4; i < QI * 4; ++i) m4[i % 4] = fmaxf(m4[i % 4], z[i]);
                    float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                    m = fmaxf(m, __shfl_xor(m, 16));
                    m = fmaxf(m, __shfl_xor(m, 32));
                    const float ms = m == -INFINITY ? 0.f : m;   // a part that lies behind the vocabulary: a sum of 0
#pragma unroll
                    for (int i = 0; i < QI * 4; ++i) s4[i % 4] += exp_of<PRECISE>(z[i] - ms);
                    float s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
                    s += __shfl_xor(s, 16);
                    s += __shfl_xor(s, 32);
                    if (fk == 0) sm[wq * BR + wr * TR + j * 16 + fl] = make_float2(m, s);
                    __builtin_amdgcn_sched_barrier(0);           // (rows in turn: all at once would not fit the registers)
                }
                lds_barrier();
                for (int r = tid; r < BR; r += NT) {
                    float2 a = sm[r];
#pragma unroll
                    for (int w = 1; w < WQ; ++w) {
                        const float2 b = sm[w * BR + r];
                        const float m = fmaxf(a.x, b.x), ms = m == -INFINITY ? 0.f : m;
                        a = make_float2(m, a.y * expf(a.x - ms) + b.y * expf(b.x - ms));
                    }
                    p.part[t.c0 / BQ * p.part_ld + t.r0 + r] = a;
                }
            } else {
                // Through LDS, 32 rows of each of the WR parts at a time (16 where there are three pieces of each value to hold): whole
                // rows of the tile are written out.
                constexpr int SLOTS = BQ / 8, pieces = PRECISE ? 3 : 1, JS = PRECISE ? 1 : 2;
                auto at = [](int row, int slot) { return row * BQ + ((slot ^ (row & 15)) << 3); };
                float lse[RI], fac[RI];
                int tgt[RI];
#pragma unroll
                for (int j = 0; j < RI; ++j) {
                    const long long row = wr0 + j * 16 + fl;
                    const bool in = row < live;
                    lse[j] = in ? p.lse[row] : 0.f;
                    fac[j] = in ? (p.grad_out ? p.grad_out[p.rowmap[row]] : 1.f) : 0.f;
                    tgt[j] = in ? p.tgt[row] : -1;
                }
                each<0, RI, JS>([&](auto at_j) {
                    constexpr int jj = decltype(at_j)::value;
                    float g[JS][QI * 4];
#pragma unroll
                    for (int j = 0; j < JS; ++j) {
                        const unsigned place = (unsigned)(tgt[jj + j] - word0);      // the target's, if it is the lane's
                        logits(jj + j, g[j]);
#pragma unroll
                        for (int i = 0; i < QI * 4; ++i) g[j][i] = exp_of<PRECISE>(g[j][i] - lse[jj + j]);
                        if (place < (unsigned)TQ && (place & 12) == 0) {
#pragma unroll
                            for (int i = 0; i < QI * 4; ++i) g[j][i] -= place == (unsigned)(i / 4 * 16 + i % 4) ? 1.f : 0.f;
                        }
                        if (edge) {
#pragma unroll
                            for (int i = 0; i < QI * 4; ++i)
                                if (i / 4 * 16 + i % 4 >= words) g[j][i] = 0.f;
                        }
#pragma unroll
                        for (int i = 0; i < QI * 4; ++i) g[j][i] *= fac[jj + j];
                        if (t.r0 + BR > live) {                  // rows behind are zeros for dW's product, whatever a word holds (0 times an infinity is none)
                            const bool in = wr0 + (jj + j) * 16 + fl < live;
#pragma unroll
                            for (int i = 0; i < QI * 4; ++i) g[j][i] = in ? g[j][i] : 0.f;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    each<0, pieces, 1>([&](auto at_piece) {
                        constexpr int piece = decltype(at_piece)::value;
#pragma unroll
                        for (int j = 0; j < JS; ++j)
#pragma unroll
                            for (int i = 0; i < QI; ++i) {
                                bf16x4 q;
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    q[e] = (bf16_t)g[j][i * 4 + e];
                                    if (piece + 1 < pieces) g[j][i * 4 + e] -= (float)q[e];      // exact; what the next piece takes
                                }
                                const int lrow = wr * 16 * JS + j * 16 + fl, col = wq * TQ + i * 16 + fk * 4;
                                *reinterpret_cast<bf16x4*>(scratch + at(lrow, col >> 3) + (col & 4)) = q;
                            }
                        lds_barrier();
                        for (int i = tid; i < WR * 16 * JS * SLOTS; i += NT) {
                            const int lrow = i / SLOTS, slot = i % SLOTS;
                            const long long row = t.r0 + lrow / (16 * JS) * TR + jj * 16 + lrow % (16 * JS);
                            *reinterpret_cast<bf16x8*>(p.g + piece * p.g_plane + row * p.g_ld + t.c0 + slot * 8) =
                                *reinterpret_cast<const bf16x8*>(scratch + at(lrow, slot));
                        }
                        lds_barrier();
                    });
                });
            }
        } else {
            // Through LDS too, as many rows at a time as it holds: a wavefront then writes whole rows of the tile.  (From the
            // registers it would write 32 or 64 bytes of sixteen rows at a time, at 1.6 TB/s.)
            if (END == STORE && p.out_bf16) {
                write_out<bf16_t, BR, BQ, WR, WQ>(scratch, static_cast<bf16_t*>(p.out), p, t.r0, t.c0, live, f, value);
            } else {
                float* out = static_cast<float*>(p.out) + (long long)t.split * ts.tiles_r * BR * p.out_ld;
                write_out<float, BR, BQ, WR, WQ>(scratch, out, p, t.r0, t.c0, live, f, value);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // (requests with empty descriptors may still be out)
}

// ---- joins -------------------------------------------------------------------------------------------------------------------
// 16 rows to a workgroup, 64 lanes to a row: a few loads in turn for any vocabulary (391 tiles: 7 us; 64 rows to a workgroup,
// 16 lanes to a row, took 14)
struct MaxSum {
    float m, sum;
    __device__ __forceinline__ void take(float2 q) {
        const float n = q.x > m ? q.x : m, ns = n == -INFINITY ? 0.f : n;
        sum = sum * expf(m - ns) + q.y * expf(q.x - ns);
        m = n;
    }
};
__global__ __launch_bounds__(1024) void join_stats_k(const float2* __restrict__ part, long long part_ld, int tiles, State s,
                                                     const float* __restrict__ target_logit, int reduction, float* __restrict__ loss,
                                                     float* __restrict__ row_loss) {
    __shared__ float2 sm[16][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, count = *s.count;
    if ((int)(blockIdx.x * 16) >= count) return;
    const int row = blockIdx.x * 16 + (lane & 15);
    MaxSum a{-INFINITY, 0.f};
#pragma unroll 4
    for (int t = wave * 4 + (lane >> 4); t < tiles; t += 64) a.take(part[t * part_ld + row]);
    a.take(make_float2(__shfl_xor(a.m, 16), __shfl_xor(a.sum, 16)));
    a.take(make_float2(__shfl_xor(a.m, 32), __shfl_xor(a.sum, 32)));
    if (lane < 16) sm[wave][lane] = make_float2(a.m, a.sum);
    __syncthreads();
    if (threadIdx.x >= 16 || row >= count) return;
    for (int w = 1; w < 16; ++w) a.take(sm[w][lane]);
    const float m = a.m, sum = a.sum;
    const bool known = s.tgt[row] >= 0;
    const float lse = known ? m + logf(sum) : NAN;
    s.lse[row] = lse;
    const float l = known ? lse - target_logit[row] : NAN;
    if (reduction == S2AG_LCE_NONE) loss[s.rowmap[row]] = l;
    else row_loss[row] = l;
}

__global__ __launch_bounds__(1024) void sum_loss_k(const float* __restrict__ row_loss, const int* __restrict__ count, int reduction,
                                                   float* __restrict__ loss) {
    __shared__ double sm[16];
    const int n = *count;
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) s += (double)row_loss[i];
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 16; ++w) s += sm[w];
    *loss = (float)(reduction == S2AG_LCE_MEAN ? s / (n > 0 ? n : 1) : s);
}

// out[r] = factor * sum over the splits: rows of dX, found by their packed place and zeros where they were ignored, or rows of dW.
// Many splits of few values go over the four wavefronts of a workgroup (136 x 300 in 85 splits: 6.2 us; a thread to each four
// columns 8.3; but 1999 x 520 11 and 8.5).
struct Finish {
    const float* acc;
    long long ld;
    int tile, tiles_q, most, slots;     // of the product
    const int *count, *inv;             // packed rows and their places; null: every row is its own
    const float* scale;                 // or null; over the number of rows that count with `mean`
    int mean;
    const int* kept;                    // that number
    long long rows;
    int dim, add;
    void* out;
};
template <typename T>
__global__ __launch_bounds__(256) void finish_k(Finish p) {
    __shared__ f32x4 sm[4][64];
    const float f = p.scale ? scale_of(p.scale, p.mean, *p.kept) : 1.f;
    const int groups = (p.dim + 3) / 4, tiles_r = ((p.count ? *p.count : (int)p.rows) + p.tile - 1) / p.tile;
    const int splits = splits_of(tiles_r * p.tiles_q, p.most, p.slots);
    const long long split = (long long)tiles_r * p.tile * p.ld;
    const long long total = p.rows * groups;
    const bool spread = splits > 8 && total <= 65536;            // (the same for every workgroup)
    const int items = spread ? 64 : 256, first = spread ? threadIdx.x >> 6 : 0, step = spread ? 4 : 1;
    const int mine = threadIdx.x & (items - 1);
    for (long long i0 = (long long)blockIdx.x * items; i0 < total; i0 += (long long)gridDim.x * items) {
        const long long i = i0 + mine, r = i / groups;
        const int c = (int)(i - r * groups) * 4;
        const long long at = i >= total ? -1 : p.inv ? (long long)p.inv[r] : r;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        if (at >= 0) {
            const float* q = p.acc + at * p.ld + c;
            int k = first;
            for (; k + 7 * step < splits; k += 8 * step) {       // eight loads in flight
                f32x4 v[8];
                for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const f32x4*>(q + (k + u * step) * split);
                for (int u = 0; u < 8; ++u) x += v[u];
            }
            for (; k < splits; k += step) x += *reinterpret_cast<const f32x4*>(q + k * split);
        }
        if (spread) {
            sm[first][mine] = x;
            __syncthreads();
            if (first == 0)
                for (int w = 1; w < 4; ++w) x += sm[w][mine];
            __syncthreads();
        }
        if (first || i >= total) continue;
        if (at >= 0) x *= f;                                     // (an infinite factor does not reach a row that was ignored)
        T* o = static_cast<T*>(p.out) + r * p.dim + c;
        for (int e = 0; e < 4; ++e)
            if (c + e < p.dim) o[e] = (T)(p.add ? (float)o[e] + x[e] : x[e]);
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------
struct Plan {
    int planes;
    long long np, vp;                   // rows and words, padded
    int kp;
    bool pack_w;
    // bytes from the state's start (kept) or the workspace's
    long long xp, wp, xh, wh, x_power, w_power;
    bool kept;
    // bytes from the workspace's start
    long long part, tl, row_loss, acc, g, dw, bytes, state_bytes;
    long long piece;                    // words of a piece of the vocabulary
    int acc_tile, splits, acc_ld;       // of the product that dX is
};

// Values of G in a piece of the vocabulary, 512 MB in bf16.  (Half as many: 8192 rows, 131072 words of 2048 values 13.0 against
// 12.8 ms; fp32, 4352 rows, 85 % of them ignored, 20000 words of 300 values: 295 against 246 us, since pieces are made for all rows.)
constexpr long long PIECE_VALUES = 1LL << 28;

bool valid(const s2ag_lce_args* a) {
    // 2^21: a tile's rows stay within a 31-bit byte offset whichever way they run
    return a && a->rows >= 0 && a->rows <= (1 << 21) && a->vocab > 0 && a->vocab <= (1 << 21) && a->dim > 0 && a->dim <= (1 << 20) &&
           a->ldx >= a->dim && a->ldw >= a->dim && a->reduction >= 0 && a->reduction <= 2 && !(a->bf16 && a->dw_accumulate);
}

constexpr int SLOTS = 256;              // large tiles: one workgroup on a compute unit; small ones: two
constexpr int small_slots = 2 * SLOTS;

// Tiles of 256 x 256 or, at `percent` of their rate, of 128 x 128.  Large ones come in rounds of one on each of the 256 compute
// units; the small ones pad less and leave less of a round idle, since half a unit's work is a finer measure.
bool big_tiles(long long r, long long q, int percent) {
    const long long big = (long long)cdiv(r, 256) * cdiv(q, 256), small = (long long)cdiv(r, 128) * cdiv(q, 128);
    return (big + SLOTS - 1) / SLOTS * (2 * small_slots) * percent <= small * 100;
}
// (bf16, 4096 rows and 32768 words of 1024 values: max and sum 281 us large, 321 small, G 306 and 320; dW 250 and 312, but of 640
// values, which large tiles pad to 768, 226 and 191)
constexpr int LOGIT_RATE = 88, DW_RATE = 77;
// Logits of short rows: a tile's end is long beside its products, and of two workgroups on a compute unit one multiplies while the
// other ends (bf16, the same rows, 320 wide: max and sum 131 us large, 129 small; 128 wide 92 and 85; fp32, 20000 words, 320 wide 238
// and 226, 1024 wide 551 and 568).  G of fp32, three pieces of each value, takes small ones for every length (320 wide: 330 and
// 291 us, 1024 wide 639 and 622).
bool short_rows(int k) { return k <= 320; }
// dX, whose words are split until the card is full (bf16, 4096 x 1024, 64 large tiles: 244 us large, 310 small; 1999 x 520, 24 of
// them: 148 and 139)
bool big_dx_tiles(long long rows, long long dim) { return (long long)cdiv(rows, 256) * cdiv(dim, 256) >= 48; }

// dW of few words and columns: the rows are split until the card is full, down to eight stages each (fp32, 8192 rows, 2000 words
// of 256 values: 65 us with the launch that joins them, in one part 417; 4096 rows, 20000 words of 128: 165 and 280).  Two parts are
// not worth that launch (bf16, 4096 rows, 10000 words of 320: 47 and 45).
int dw_splits(long long words, int dim, long long rows, int products) {
    if (big_tiles(words, dim, DW_RATE)) return 1;
    const long long tiles = (long long)cdiv(words, 128) * cdiv(dim, 128), stages = rows / BK * products;
    const long long splits = std::min(small_slots / tiles, stages / 8);
    return splits < 3 ? 1 : (int)splits;
}

Plan plan(const s2ag_lce_args* a, bool backward) {
    Plan p{};
    p.planes = a->bf16 ? 1 : 3;
    p.np = padded(a->rows);
    p.vp = round_up(a->vocab, 256);
    p.kp = (int)round_up(a->dim, BK);
    p.pack_w = !(a->bf16 && a->dim % BK == 0 && a->ldw % 8 == 0 && a->ldw <= (1 << 21) && aligned16(a->w));
    long long at = 0;
    auto take = [&](long long b) {
        const long long here = at;
        at += round_up(b, 256);
        return here;
    };
    p.kept = backward || a->keep;
    long long kept_bytes = round_up(4 * state_words(a->rows), 256);
    auto put = [&](long long b) {                                 // into the state, if that is kept
        if (!p.kept) return take(b);
        const long long here = kept_bytes;
        kept_bytes += round_up(b, 256);
        return here;
    };
    if (!a->bf16) {
        p.xh = put(2 * 2 * p.np * p.kp);
        p.wh = put(2 * 2 * a->vocab * p.kp);
        p.x_power = put(4 * p.np);
        p.w_power = put(4 * p.vp);
    }
    if (a->bf16 || p.kept) {                                      // (the pieces are the gradient's)
        p.xp = put(2 * p.planes * p.np * p.kp);
        p.wp = p.pack_w ? put(2 * p.planes * a->vocab * p.kp) : 0;
    }
    p.state_bytes = kept_bytes;
    if (!backward) {
        p.part = take(8 * p.np * cdiv(a->vocab, 128));
        p.tl = take(4 * p.np);
        p.row_loss = take(4 * p.np);
    } else {
        const long long most = PIECE_VALUES / p.planes / (p.np ? p.np : 1) / 256 * 256;
        const long long pieces = cdiv(p.vp, most < 1024 ? 1024 : most);
        p.piece = round_up(cdiv(p.vp, pieces), 256);
        const bool dx = a->dx != nullptr;
        p.acc_ld = (int)round_up(a->dim, 4);
        // dX has few tiles: the words of a piece are split, down to eight stages each
        p.acc_tile = big_dx_tiles(p.np, a->dim) ? 256 : 128;
        const long long stages = p.piece / BK * (a->bf16 ? 1 : 6);
        p.splits = (int)(stages / 8 < 1 ? 1 : stages / 8 > small_slots ? small_slots : stages / 8);
        // (what fills the card with splits is no more than its tiles hold)
        p.acc = take(dx ? 4 * (p.np * p.acc_ld + (long long)SLOTS * 256 * 256) : 0);
        p.g = take(2 * p.planes * p.np * p.piece);
        // (splits that fill the card are no more than its tiles hold; the last piece may be split where the others are not)
        const long long last = a->vocab - (p.vp - 1) / p.piece * p.piece;
        const bool split = dw_splits(last < p.piece ? last : p.piece, a->dim, p.np, a->bf16 ? 1 : 6) > 1;
        p.dw = take(a->dw && split ? 4LL * small_slots * 128 * 128 : 0);
    }
    p.bytes = at;
    return p;
}

template <int BR, int BQ, int WR, int WQ, End END, bool PRECISE>
int launch_tiles(Product& p, long long r_rows, long long q_rows, hipStream_t st) {
    constexpr int LDS = (2 * (BR + BQ) * BK + 64 * BQ) * 2, PER_CU = BR == 256 ? 1 : 2;
    static_assert(LDS * PER_CU <= 160 * 1024 && WR == 2 && 64 * BQ * 2 >= WQ * BR * 8, "the ends' scratch");
    // (every time: the attribute belongs to the current device)
    if (hipFuncSetAttribute((const void*)product_k<BR, BQ, WR, WQ, END, PRECISE>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
        return S2AG_E_UNSUPPORTED;
    p.tiles_q = cdiv(q_rows, BQ);
    p.slots = SLOTS * PER_CU;
    if (p.splits < 1) p.splits = 1;
    if ((long long)cdiv(r_rows, BR) * p.tiles_q * p.splits > 0x3fffffffLL) return S2AG_E_UNSUPPORTED;
    if (r_rows == 0 || q_rows == 0) return 0;
    hipLaunchKernelGGL((product_k<BR, BQ, WR, WQ, END, PRECISE>), dim3(p.slots), dim3(64 * WR * WQ), LDS, st, p);
    S2AG_LAUNCH_CHECK();
    return 0;
}

template <End END>
int launch(Product& p, bool big, long long r_rows, long long q_rows, hipStream_t st) {
    if constexpr (END == GRADS) {
        if (p.fp32) return launch_tiles<128, 128, 2, 2, END, true>(p, r_rows, q_rows, st);
    } else {
        if (p.fp32) return big ? launch_tiles<256, 256, 2, 2, END, true>(p, r_rows, q_rows, st) : launch_tiles<128, 128, 2, 2, END, true>(p, r_rows, q_rows, st);
    }
    return big ? launch_tiles<256, 256, 2, 2, END, false>(p, r_rows, q_rows, st) : launch_tiles<128, 128, 2, 2, END, false>(p, r_rows, q_rows, st);
}

unsigned grid_of(long long work, int block = 256) {
    const long long b = (work + block - 1) / block, most = 4096 * 256 / block;
    return (unsigned)(b < 1 ? 1 : b > most ? most : b);
}
template <typename T> long long packers(int kp) { return sizeof(T) == 4 ? 64 : kp / 8; }      // threads to a row

// where the packed operands are, or the caller's W as it is
char* packed(const s2ag_lce_args* a, const Plan& p) { return static_cast<char*>(p.kept ? a->state : a->workspace); }
void operands(const s2ag_lce_args* a, const Plan& p, Operand* x, Operand* w) {
    *x = Operand{reinterpret_cast<bf16_t*>(packed(a, p) + p.xp), p.np * p.kp, p.kp};
    if (p.pack_w) *w = Operand{reinterpret_cast<bf16_t*>(packed(a, p) + p.wp), a->vocab * p.kp, p.kp};
    else *w = Operand{static_cast<const bf16_t*>(a->w), 0, a->ldw};
}
// those of the logits from word v0 on
void logit_operands(const s2ag_lce_args* a, const Plan& p, long long v0, Product* q) {
    if (a->bf16) {
        operands(a, p, &q->r, &q->q);
    } else {
        q->r = Operand{reinterpret_cast<bf16_t*>(packed(a, p) + p.xh), p.np * p.kp, p.kp};
        q->q = Operand{reinterpret_cast<bf16_t*>(packed(a, p) + p.wh), a->vocab * p.kp, p.kp};
        q->r_power = reinterpret_cast<int*>(packed(a, p) + p.x_power);
        q->q_power = reinterpret_cast<int*>(packed(a, p) + p.w_power) + v0;
    }
    q->q.p += v0 * q->q.ld;
    q->r_rows = p.np;
    q->k = p.kp;
    q->fp32 = !a->bf16;
}

template <typename T>
int pack(const s2ag_lce_args* a, const Plan& p, const Select& s, Pack<T> x, Pack<T> w, hipStream_t st) {
    x.src = static_cast<const T*>(a->x);
    x.ld = a->ldx;
    x.rows = p.np;
    x.rowmap = s.s.rowmap;
    x.count = s.s.count;
    w.src = static_cast<const T*>(a->w);
    w.ld = a->ldw;
    w.rows = a->vocab;
    x.dim = w.dim = a->dim;
    x.kp = w.kp = p.kp;
    if (p.pack_w)
        hipLaunchKernelGGL(select_and_pack_k<T>, dim3(1 + grid_of(a->vocab * packers<T>(p.kp), 1024)), dim3(1024), 0, st, s, w);
    else
        hipLaunchKernelGGL(select_rows_k, dim3(1), dim3(1024), 0, st, s);
    S2AG_LAUNCH_CHECK();
    hipLaunchKernelGGL(pack_k<T>, dim3(grid_of(p.np * packers<T>(p.kp), 256)), dim3(256), 0, st, x);
    S2AG_LAUNCH_CHECK();
    return 0;
}
int select_and_pack(const s2ag_lce_args* a, const Plan& p, const Select& s, hipStream_t st) {
    char* at = packed(a, p);
    if (a->bf16) {
        Pack<bf16_t> x{}, w{};
        x.dst = reinterpret_cast<bf16_t*>(at + p.xp);
        w.dst = reinterpret_cast<bf16_t*>(at + p.wp);
        return pack(a, p, s, x, w, st);
    }
    Pack<float> x{}, w{};
    x.halves = reinterpret_cast<f16_t*>(at + p.xh);
    w.halves = reinterpret_cast<f16_t*>(at + p.wh);
    x.power = reinterpret_cast<int*>(at + p.x_power);
    w.power = reinterpret_cast<int*>(at + p.w_power);
    if (p.kept) {
        x.pieces = reinterpret_cast<bf16_t*>(at + p.xp);
        w.pieces = reinterpret_cast<bf16_t*>(at + p.wp);
    }
    x.plane = p.np * p.kp;
    w.plane = a->vocab * p.kp;
    return pack(a, p, s, x, w, st);
}

int finish(const s2ag_lce_args* a, Finish& e, hipStream_t st) {
    e.dim = a->dim;
    const dim3 grid(grid_of(e.rows * ((a->dim + 3) / 4) * 4));
    if (a->bf16) hipLaunchKernelGGL(finish_k<bf16_t>, grid, dim3(256), 0, st, e);
    else hipLaunchKernelGGL(finish_k<float>, grid, dim3(256), 0, st, e);
    S2AG_LAUNCH_CHECK();
    return 0;
}
bool ready(const s2ag_lce_args* a, const Plan& p) {
    return a->x && a->w && a->target && a->state && a->workspace && a->workspace_bytes >= p.bytes && aligned16(a->workspace) && aligned16(a->state);
}
}  // namespace

extern "C" long long s2ag_lce_state_bytes(const s2ag_lce_args* a) {
    if (!valid(a)) return S2AG_E_BADARG;
    return plan(a, false).state_bytes;
}

extern "C" long long s2ag_lce_workspace_bytes(const s2ag_lce_args* a, int backward) {
    if (!valid(a)) return S2AG_E_BADARG;
    return plan(a, backward != 0).bytes + 256;
}

extern "C" int s2ag_lce_fwd(const s2ag_lce_args* a, void* stream) {
    if (!valid(a)) return S2AG_E_BADARG;
    hipStream_t st = (hipStream_t)stream;
    const Plan p = plan(a, false);
    if (!a->loss || (a->rows && !ready(a, p)) || !a->state) return S2AG_E_BADARG;
    const State s = state_of(a->state, a->rows);
    char* ws = static_cast<char*>(a->workspace);
    float* row_loss = reinterpret_cast<float*>(ws + p.row_loss);
    const Select sel{a->target, a->target_i32, a->rows, a->vocab, a->ignore_index, s, a->reduction == S2AG_LCE_NONE ? a->loss : nullptr};
    if (a->rows == 0) {
        hipLaunchKernelGGL(select_rows_k, dim3(1), dim3(1024), 0, st, sel);
        S2AG_LAUNCH_CHECK();
    } else {
        Product q{};
        if (int rc = select_and_pack(a, p, sel, st)) return rc;
        logit_operands(a, p, 0, &q);
        q.q_rows = q.vocab = a->vocab;
        q.r_count = s.count;
        q.tgt = s.tgt;
        q.part = reinterpret_cast<float2*>(ws + p.part);
        q.part_ld = p.np;
        q.target_logit = reinterpret_cast<float*>(ws + p.tl);
        if (int rc = launch<STATS>(q, !short_rows(p.kp) && big_tiles(p.np, a->vocab, LOGIT_RATE), p.np, a->vocab, st)) return rc;
        hipLaunchKernelGGL(join_stats_k, dim3((unsigned)(p.np / 16)), dim3(1024), 0, st, q.part, q.part_ld, q.tiles_q, s, q.target_logit,
                           a->reduction, a->loss, row_loss);
        S2AG_LAUNCH_CHECK();
    }
    if (a->reduction != S2AG_LCE_NONE) {
        hipLaunchKernelGGL(sum_loss_k, dim3(1), dim3(1024), 0, st, row_loss, s.count, a->reduction, a->loss);
        S2AG_LAUNCH_CHECK();
    }
    return 0;
}

extern "C" int s2ag_lce_bwd(const s2ag_lce_args* a, void* stream) {
    if (!valid(a)) return S2AG_E_BADARG;
    hipStream_t st = (hipStream_t)stream;
    const Plan p = plan(a, true);
    if (!a->grad_out || !ready(a, p)) return S2AG_E_BADARG;
    if (!a->dx && !a->dw) return 0;
    const State s = state_of(a->state, a->rows);
    char* ws = static_cast<char*>(a->workspace);
    const bool each = a->reduction == S2AG_LCE_NONE, mean = a->reduction == S2AG_LCE_MEAN;
    Operand x, w;
    operands(a, p, &x, &w);
    bf16_t* g = reinterpret_cast<bf16_t*>(ws + p.g);
    float* acc = reinterpret_cast<float*>(ws + p.acc);
    for (long long v0 = 0; v0 < p.vp; v0 += p.piece) {
        const long long words = a->vocab - v0 < p.piece ? a->vocab - v0 : p.piece;     // that exist
        if (words <= 0) break;
        const long long wide = round_up(words, 256);
        Product q{};
        logit_operands(a, p, v0, &q);
        q.q_rows = words;
        q.r_count = s.count;
        q.tgt = s.tgt;
        q.q0 = v0;
        q.vocab = a->vocab;
        q.lse = s.lse;
        q.grad_out = each ? a->grad_out : nullptr;
        q.rowmap = s.rowmap;
        q.g = g;
        q.g_ld = p.piece;
        q.g_plane = p.np * p.piece;
        if (int rc = launch<GRADS>(q, !short_rows(p.kp) && big_tiles(p.np, wide, LOGIT_RATE), p.np, wide, st)) return rc;
        if (a->dx) {
            Product d{};
            d.r = Operand{g, q.g_plane, p.piece};
            d.q = Operand{w.p + v0 * w.ld, w.plane, w.ld};
            d.r_rows = p.np;
            d.q_rows = d.cols = a->dim;
            d.q_deep = words;
            d.q_cols = p.pack_w ? p.kp : a->dim;
            d.k = (int)wide;
            d.fp32 = !a->bf16;
            d.r_count = s.count;
            d.splits = p.splits;
            d.out = acc;
            d.out_ld = p.acc_ld;
            d.add = v0 > 0;
            if (int rc = launch<ACCUM>(d, p.acc_tile == 256, p.np, a->dim, st)) return rc;
        }
        if (a->dw) {
            Product d{};
            d.r = Operand{g, q.g_plane, p.piece};
            d.q = x;
            d.r_rows = words;
            d.q_rows = d.cols = a->dim;
            d.r_deep = d.q_deep = p.np;
            d.r_cols = (int)p.piece;
            d.q_cols = p.kp;
            d.k_count = s.count;
            d.fp32 = !a->bf16;
            void* dw = a->bf16 ? (void*)(static_cast<bf16_t*>(a->dw) + v0 * a->dim) : (void*)(static_cast<float*>(a->dw) + v0 * a->dim);
            d.splits = dw_splits(words, a->dim, p.np, a->bf16 ? 1 : 6);
            if (d.splits > 1) {
                Finish e{};
                e.most = d.splits;
                d.out = ws + p.dw;
                d.out_ld = p.acc_ld;
                if (int rc = launch<STORE>(d, false, words, a->dim, st)) return rc;
                e.acc = reinterpret_cast<const float*>(ws + p.dw);
                e.ld = p.acc_ld;
                e.tile = 128;
                e.tiles_q = cdiv(a->dim, 128);
                e.slots = small_slots;
                e.scale = each ? nullptr : a->grad_out;
                e.mean = mean;
                e.kept = s.count;
                e.rows = words;
                e.add = a->dw_accumulate;
                e.out = dw;
                if (int rc = finish(a, e, st)) return rc;
                continue;
            }
            d.out = dw;
            d.out_ld = a->dim;
            d.out_bf16 = a->bf16;
            d.add = a->dw_accumulate;
            d.scale = each ? nullptr : a->grad_out;
            d.mean = mean;
            if (int rc = launch<STORE>(d, big_tiles(words, a->dim, DW_RATE), words, a->dim, st)) return rc;
        }
    }
    if (a->dx && a->rows) {
        Finish e{};
        e.acc = acc;
        e.ld = p.acc_ld;
        e.tile = p.acc_tile;
        e.tiles_q = cdiv(a->dim, p.acc_tile);
        e.most = p.splits;
        e.slots = p.acc_tile == 256 ? SLOTS : small_slots;
        e.count = s.count;
        e.inv = s.inv;
        e.scale = each ? nullptr : a->grad_out;
        e.mean = mean;
        e.kept = s.count;
        e.rows = a->rows;
        e.out = a->dx;
        if (int rc = finish(a, e, st)) return rc;
    }
    return 0;
}
