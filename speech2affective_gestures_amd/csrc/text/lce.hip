// Softmax cross entropy of a linear layer over a large vocabulary, without keeping the logits, and its gradient.
//
//   z = X W^T        loss_i = log sum_v exp z_iv - z_{i,t_i}
//   G = g_i (softmax(z)_iv - [v = t_i])        dX = G W        dW = G^T X
//
// Bound by the matrix pipe: 2 N V D operations for the loss, 8 N V D with the gradient (the logits are formed twice: keeping
// them would be N V values, the largest tensor of a training step by far).
//
// All four products are ONE tiled product out[r][c] = sum_k R[r][k] Q[c][k] of two bf16 matrices whose rows run along k, with
// four ends: (1) max and sum of exponentials of each row of a tile of logits, joined over the tiles by a small launch;
// (2) G of a piece of the vocabulary, stored as [row][word] and as [word][row]; (3) dX += G W over that piece in fp32;
// (4) dW of that piece.  Operands whose rows do not run along k are transposed once (X^T, W^T: small beside the products).
//
// The rows that are ignored are left out of every product: the others are packed in front (rowmap), their number stays on the
// device, and the tiles behind it end at once.
//
// fp32 operands are taken as three bf16 pieces (v = p0 + p1 + p2 to 2^-25) and the six products of pieces that matter at fp32's
// own rounding: still more than twice the rate of the f32 matrix instructions.  bf16 operands need one product; there G is
// rounded to bf16 (2^-9 of each value; sums stay in fp32), without its factor g where that is one number for all rows.
#include "text_common.h"

namespace {
using namespace s2ag;
using namespace s2ag::text;

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
__global__ __launch_bounds__(1024) void select_rows_k(const void* __restrict__ target, int i32, long long rows, long long vocab,
                                                      long long ignore, State s, float* loss_rows) {
    __shared__ int sm[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int base = 0;
    for (long long r0 = 0; r0 < rows; r0 += 1024) {
        const long long r = r0 + threadIdx.x;
        const long long t = r < rows ? load_id(target, i32, r) : ignore;
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
            if (loss_rows && !keep) loss_rows[r] = 0.f;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) *s.count = base;
}

// ---- operands: rows along k, padded with zeros to a multiple of 64, fp32 as three bf16 pieces --------------------------------
struct Operand {
    const bf16_t* p;
    long long plane, ld;                // elements
};

__device__ __forceinline__ void split3(float v, bf16_t* q) {
    q[0] = (bf16_t)v;
    const float r1 = v - (float)q[0];   // exact
    q[1] = (bf16_t)r1;
    q[2] = (bf16_t)(r1 - (float)q[1]);
}

// dst[r][0..kp) from row rowmap[r] (or r) of src, zeros behind column dim and for r >= count (up to `rows`).  An infinity
// leaves NaN in the second piece, as its products would anyway.
template <typename T>
__global__ __launch_bounds__(256) void pack_k(const T* __restrict__ src, long long ld, int dim, const int* __restrict__ rowmap,
                                              const int* __restrict__ count, long long rows, bf16_t* __restrict__ dst, int kp,
                                              long long plane) {
    const long long live = count ? (long long)*count : rows;
    const long long end = count ? (live + ROWS - 1) / ROWS * ROWS : rows;
    const int groups = kp / 8;
    const long long total = end * groups;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / groups;
        const int c = (int)(i - r * groups) * 8;
        const bool in = r < live;
        const T* s = src + (in ? (rowmap ? (long long)rowmap[r] : r) : 0) * ld;
        bf16x8 q[3];
        for (int j = 0; j < 8; ++j) {
            const float v = in && c + j < dim ? (float)s[c + j] : 0.f;
            if constexpr (sizeof(T) == 2) {
                q[0][j] = (bf16_t)v;
            } else {
                bf16_t p[3];
                split3(v, p);
                for (int k = 0; k < 3; ++k) q[k][j] = p[k];
            }
        }
        for (int k = 0; k < (sizeof(T) == 2 ? 1 : 3); ++k) *reinterpret_cast<bf16x8*>(dst + k * plane + r * kp + c) = q[k];
    }
}

// dst[c][r] = src[r][c] for r < rows (zeros behind, up to the multiple of 64 that holds rows_end), c < cols; 64 x 64 a workgroup
__global__ __launch_bounds__(256) void transpose_k(Operand src, long long rows, const int* __restrict__ count, int cols,
                                                   bf16_t* __restrict__ dst, long long ld_dst, long long plane_dst) {
    __shared__ bf16_t sm[64][66];
    const long long r0 = (long long)blockIdx.x * 64;
    const int c0 = blockIdx.y * 64;
    if (count && r0 >= (long long)*count) return;                // (packed rows are zero up to a multiple of 256)
    const bf16_t* s = src.p + blockIdx.z * src.plane;
    bf16_t* d = dst + blockIdx.z * plane_dst;
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
        const int r = i >> 6, c = i & 63;
        sm[r][c] = r0 + r < rows && c0 + c < cols ? s[(r0 + r) * src.ld + c0 + c] : (bf16_t)0.f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 8; i += 256) {
        const int c = i >> 3, r = (i & 7) * 8;
        if (c0 + c >= cols) continue;
        bf16x8 q;
        for (int j = 0; j < 8; ++j) q[j] = sm[r + j][c];
        *reinterpret_cast<bf16x8*>(d + (long long)(c0 + c) * ld_dst + r0 + r) = q;
    }
}

// ---- the tiled product -------------------------------------------------------------------------------------------------------
enum End { STATS, GRADS, ACCUM, STORE };

struct Product {
    Operand r, q;
    long long r_rows, q_rows;           // rows that exist
    int k;                              // of one pair of pieces, a multiple of 64
    const int* k_count;                 // not null: k is this, rounded up to 64
    const int* r_count;                 // not null: rows of R that matter
    int pairs;                          // 1, or 6 of three pieces
    int tiles_r, tiles_q, splits;
    // STATS: max and sum of exponentials [tile_q][padded rows], logit of the target; GRADS: lse, factor of each row
    const int* tgt;
    long long q0;                       // word number of Q's first row
    long long vocab;
    float2* part;
    long long part_ld;
    float* target_logit;
    const float *lse, *factor;
    bf16_t *g, *gt;                     // GRADS: [row][word] pitch g_ld, [word][row] pitch gt_ld (either may be null)
    long long g_ld, g_plane, gt_ld, gt_plane;
    // ACCUM: fp32 [split][row][col] pitch out_ld; STORE: rows of dW
    void* out;
    long long out_ld, out_split;
    int cols, add, out_bf16;
    const float* scale;                 // STORE: the factor of all rows
};

// pairs of pieces, the smallest products first: (0, 2) (1, 1) (2, 0) (0, 1) (1, 0) (0, 0), two bits each
__device__ __forceinline__ int piece_r(int pair) { return (0x124 >> (2 * pair)) & 3; }
__device__ __forceinline__ int piece_q(int pair) { return (0x046 >> (2 * pair)) & 3; }

typedef short s16x4_t __attribute__((ext_vector_type(4)));
#define S2AG_LDS_PTR(type, p) ((__attribute__((address_space(3))) type*)(p))

// 16-byte slot of (row, slot) in a stage: the slots of a row are permuted by the row's low bits, so that the 16 rows that a
// wavefront reads at one slot lie in different banks.
__device__ __forceinline__ int slot_at(int row, int slot) { return row * BK + ((slot ^ (row & 7)) << 3); }

// 16 bytes a lane from the buffer to LDS: lane l's land at dst + 16 l
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t from, bf16_t* dst, unsigned lane_offset, int offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, S2AG_LDS_PTR(void, dst), 16, lane_offset, offset, 0, 0);
}

// Matrix instruction with its accumulator in the accumulation registers, where the compiler, left to itself, moves a set that
// fills all 256 of them to and fro.  The compiler knows no matrix instruction here: `settle` stands between the last of them
// and the first use of a result, and between the zeros and the first of them.
__device__ __forceinline__ void mfma_acc(f32x4& c, bf16x8 a, bf16x8 b) {
    asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

template <int BR, int BQ, int WR, int WQ, End END>
__global__ __launch_bounds__(64 * WR * WQ, 1) void product_k(Product p) {
    constexpr int NT = 64 * WR * WQ;
    constexpr int TR = BR / WR, TQ = BQ / WQ, RI = TR / 16, QI = TQ / 16;      // a wavefront's part
    constexpr int LR = BR * 8 / NT, LQ = BQ * 8 / NT;                          // 16-byte loads per thread and stage
    constexpr int STAGE = (BR + BQ) * BK;
    extern __shared__ __attribute__((aligned(16))) bf16_t lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave / WQ, wq = wave % WQ;

    // Workgroups are dealt to the eight XCDs in turn; the remap gives each XCD a contiguous range of tiles, and inside it the
    // tiles go column by column over GROUP row tiles, so that the tiles that run at the same time share operands in its L2.
    int v;
    {
        const int n = gridDim.x, x = blockIdx.x & 7, q8 = n >> 3, r8 = n & 7;
        v = (x < r8 ? x * (q8 + 1) : r8 * (q8 + 1) + (x - r8) * q8) + (blockIdx.x >> 3);
    }
    // (whole-number division runs on the vector units: the results are told to be one for the wavefront, so that the operands'
    // descriptors stay in scalar registers)
    const int split = __builtin_amdgcn_readfirstlane(v % p.splits);
    v = __builtin_amdgcn_readfirstlane(v / p.splits);
    constexpr int GROUP = 8;
    const int per = GROUP * p.tiles_q, grp = v / per, first = grp * GROUP;
    const int gsz = min(p.tiles_r - first, GROUP);
    const int tr = __builtin_amdgcn_readfirstlane(first + (v - grp * per) % gsz), tq = __builtin_amdgcn_readfirstlane((v - grp * per) / gsz);
    const long long r0 = (long long)tr * BR, c0 = (long long)tq * BQ;
    const long long live = p.r_count ? (long long)__builtin_amdgcn_readfirstlane(*p.r_count) : p.r_rows;
    if (r0 >= live) return;

    const int kt = p.k_count ? __builtin_amdgcn_readfirstlane((*p.k_count + BK - 1) / BK) : p.k / BK, total = kt * p.pairs;
    const int it0 = __builtin_amdgcn_readfirstlane((int)((long long)total * split / p.splits));
    const int it1 = __builtin_amdgcn_readfirstlane((int)((long long)total * (split + 1) / p.splits));

    const long long r_left = p.r_rows - r0, q_left = p.q_rows > c0 ? p.q_rows - c0 : 0;      // (a tile may lie behind the words)
    const int r_bytes = (int)((r_left < BR ? r_left : BR) * p.r.ld * 2), q_bytes = (int)((q_left < BQ ? q_left : BQ) * p.q.ld * 2);
    const int ld_row = tid >> 3, ld_slot = (tid & 7) ^ (ld_row & 7);
    unsigned r_off[LR], q_off[LQ];
#pragma unroll
    for (int i = 0; i < LR; ++i) r_off[i] = (unsigned)((ld_row + i * (NT / 8)) * p.r.ld * 2 + ld_slot * 16);
#pragma unroll
    for (int i = 0; i < LQ; ++i) q_off[i] = (unsigned)((ld_row + i * (NT / 8)) * p.q.ld * 2 + ld_slot * 16);

    // the stage that is requested next: its pair of pieces, its place along k; behind the last one the descriptors are empty, so
    // that the loop has no branch
    int pair = __builtin_amdgcn_readfirstlane(it0 / (kt > 0 ? kt : 1)), kk = it0 - pair * kt, left = it1 - it0;
    __amdgpu_buffer_rsrc_t rr, qr;
    auto descriptors = [&]() {
        const bf16_t* rb = p.r.p + piece_r(p.pairs == 1 ? 5 : pair) * p.r.plane + r0 * p.r.ld;
        const bf16_t* qb = p.q.p + piece_q(p.pairs == 1 ? 5 : pair) * p.q.plane + c0 * p.q.ld;
        rr = __builtin_amdgcn_make_buffer_rsrc((void*)rb, 0, left > 0 ? r_bytes : 0, 0x00020000);
        qr = __builtin_amdgcn_make_buffer_rsrc((void*)qb, 0, left > 0 ? q_bytes : 0, 0x00020000);
    };
    descriptors();
    // requests [from, from + n) of the LR + LQ of a stage
    auto issue = [&](int buf, int from, int n) {
        bf16_t* s = lds + buf * STAGE + wave * 512;
        const int off = kk * (BK * 2);
#pragma unroll
        for (int i = from; i < from + n; ++i) {
            if (i < LR) to_lds(rr, s + i * NT * 8, r_off[i < LR ? i : 0], off);
            else to_lds(qr, s + BR * BK + (i - LR) * NT * 8, q_off[i < LR ? 0 : i - LR], off);
        }
    };
    auto advance = [&]() {
        --left;
        if (++kk == kt) {
            kk = 0;
            pair = pair + 1 < p.pairs ? pair + 1 : pair;
        }
        descriptors();
    };

    f32x4 acc[QI][RI];
#pragma unroll
    for (int i = 0; i < QI; ++i)
#pragma unroll
        for (int j = 0; j < RI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int fl = lane & 15, fk = lane >> 4;
    const bf16_t* const rs = lds + wr * TR * BK;
    const bf16_t* const qs = lds + BR * BK + wq * TQ * BK;
    // fragment [u] of half ks of a stage: the QI of Q, then the RI of R
    auto fragment = [&](bf16x8 (&a)[QI], bf16x8 (&b)[RI], int buf, int ks, int u) {
        if (u < QI) a[u < QI ? u : 0] = *reinterpret_cast<const bf16x8*>(qs + buf * STAGE + slot_at(u * 16 + fl, ks * 4 + fk));
        else b[u < QI ? 0 : u - QI] = *reinterpret_cast<const bf16x8*>(rs + buf * STAGE + slot_at((u - QI) * 16 + fl, ks * 4 + fk));
    };
    auto multiply = [&](const bf16x8 (&a)[QI], const bf16x8 (&b)[RI], int i) {
#pragma unroll
        for (int j = 0; j < RI; ++j) {
            if constexpr (RI * QI * 4 == 256) mfma_acc(acc[i][j], a[i], b[j]);
            else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
        }
    };

    // Two stages in LDS, two halves of a stage in registers.  While the first half of a stage is multiplied its second half is
    // read; then every wavefront is done with the stage's LDS, the next stage (requested a whole stage ago) has landed, and while
    // the second half is multiplied the first half of the next stage is read and the stage after it is requested.  Reads and
    // requests go behind rows of matrix instructions, the reads behind the first ones, so that they run beside the others.
    constexpr int PER = (QI + RI + QI / 2 - 1) / (QI / 2), LPER = (LR + LQ + QI - 1) / QI;
    const int stages = it1 - it0;
    bf16x8 a0[QI], b0[RI], a1[QI], b1[RI];
    issue(0, 0, LR + LQ);
    advance();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    issue(1, 0, LR + LQ);
    advance();
#pragma unroll
    for (int u = 0; u < QI + RI; ++u) fragment(a0, b0, 0, 0, u);
    settle();
    for (int n = 0; n < stages; ++n) {
        const int buf = n & 1;
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            multiply(a0, b0, i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = i * PER; u < (i + 1) * PER && u < QI + RI; ++u) fragment(a1, b1, buf, 1, u);
            __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // (keeps the reads behind the barrier)
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            multiply(a1, b1, i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = i * PER; u < (i + 1) * PER && u < QI + RI; ++u) fragment(a0, b0, buf ^ 1, 0, u);
            issue(buf, i * LPER, (i + 1) * LPER < LR + LQ ? LPER : LR + LQ - i * LPER);
            __builtin_amdgcn_sched_barrier(0);
        }
        advance();
    }
    settle();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();

    // element e of acc[i][j]: column i * 16 + fk * 4 + e, row j * 16 + fl of the wavefront's part
    const long long wr0 = r0 + wr * TR, wc0 = c0 + wq * TQ;
    if constexpr (END == STATS) {
        float2* sm = reinterpret_cast<float2*>(lds);             // [WQ][BR]
#pragma unroll
        for (int j = 0; j < RI; ++j) {
            const long long row = wr0 + j * 16 + fl;
            const int t = row < live ? p.tgt[row] : -1;
            float m = -INFINITY;
            bool mine = false;
            float tl = 0.f;
#pragma unroll
            for (int i = 0; i < QI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const long long c = p.q0 + wc0 + i * 16 + fk * 4 + e;
                    if (c == t) {
                        tl = acc[i][j][e];
                        mine = true;
                    }
                    if (c >= p.vocab) acc[i][j][e] = -INFINITY;
                    m = fmaxf(m, acc[i][j][e]);
                }
            if (mine) p.target_logit[row] = tl;
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            const float ms = m == -INFINITY ? 0.f : m;           // a part that lies behind the vocabulary: a sum of 0
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < QI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s += p.pairs == 1 ? __expf(acc[i][j][e] - ms) : expf(acc[i][j][e] - ms);
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            if (fk == 0) sm[wq * BR + wr * TR + j * 16 + fl] = make_float2(m, s);
        }
        __syncthreads();
        for (int r = tid; r < BR; r += NT) {
            float2 a = sm[r];
#pragma unroll
            for (int w = 1; w < WQ; ++w) {
                const float2 b = sm[w * BR + r];
                const float m = fmaxf(a.x, b.x), ms = m == -INFINITY ? 0.f : m;
                a = make_float2(m, a.y * expf(a.x - ms) + b.y * expf(b.x - ms));
            }
            p.part[tq * p.part_ld + r0 + r] = a;
        }
    } else if constexpr (END == GRADS) {
        // through LDS as [row][word]: rows are written out from it as they are, columns by the transposing read
        constexpr int SLOTS = BQ / 8;
        auto at = [](int row, int slot) { return row * BQ + ((slot ^ (row & (SLOTS - 1 < 15 ? SLOTS - 1 : 15))) << 3); };
        const int pieces = p.pairs == 1 ? 1 : 3;
        for (int piece = 0; piece < pieces; ++piece) {           // (a piece is split off the value formed again: no registers for rests)
            if (piece) __syncthreads();
#pragma unroll
            for (int j = 0; j < RI; ++j) {
                const long long row = wr0 + j * 16 + fl;
                const bool in = row < live;
                const float lse = in ? p.lse[row] : 0.f, fac = in ? (p.factor ? p.factor[row] : 1.f) : 0.f;
                const int t = in ? p.tgt[row] : -1;
#pragma unroll
                for (int i = 0; i < QI; ++i) {
                    bf16x4 q;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int c = (int)(p.q0 + wc0) + i * 16 + fk * 4 + e;
                        float g = p.pairs == 1 ? __expf(acc[i][j][e] - lse) : expf(acc[i][j][e] - lse);
                        if (c == t) g -= 1.f;
                        g = in && c < (int)p.vocab ? g * fac : 0.f;
                        q[e] = (bf16_t)g;
                        if (piece) {
                            const float rest = g - (float)q[e];
                            q[e] = (bf16_t)rest;
                            if (piece == 2) q[e] = (bf16_t)(rest - (float)q[e]);
                        }
                    }
                    const int at_row = wr * TR + j * 16 + fl, col = wq * TQ + i * 16 + fk * 4;
                    *reinterpret_cast<bf16x4*>(lds + at(at_row, col >> 3) + (col & 4)) = q;
                }
                __builtin_amdgcn_sched_barrier(0);               // (rows in turn: all at once would not fit the registers)
            }
            __syncthreads();
            if (p.g)
                for (int i = tid; i < BR * SLOTS; i += NT) {
                    const int row = i / SLOTS, slot = i % SLOTS;
                    *reinterpret_cast<bf16x8*>(p.g + piece * p.g_plane + (r0 + row) * p.g_ld + c0 + slot * 8) =
                        *reinterpret_cast<const bf16x8*>(lds + at(row, slot));
                }
            if (p.gt)
                // a wavefront takes 16 words x 32 rows: its four groups of 16 lanes eight rows each, in two reads of four
                for (int u = wave; u < (BQ / 16) * (BR / 32); u += NT / 64) {
                    const int w0 = (u % (BQ / 16)) * 16, rr = (u / (BQ / 16)) * 32 + fk * 8;
                    bf16x8 q;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int row = rr + h * 4 + (fl >> 2), col = w0 + (fl & 3) * 4;
                        const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            S2AG_LDS_PTR(s16x4_t, lds + at(row, col >> 3) + (col & 4)));
                        const bf16x4 y = __builtin_bit_cast(bf16x4, x);
#pragma unroll
                        for (int e = 0; e < 4; ++e) q[h * 4 + e] = y[e];
                    }
                    *reinterpret_cast<bf16x8*>(p.gt + piece * p.gt_plane + (c0 + w0 + fl) * p.gt_ld + r0 + rr) = q;
                }
        }
    } else if constexpr (END == ACCUM) {
        float* out = static_cast<float*>(p.out) + split * p.out_split;
#pragma unroll
        for (int j = 0; j < RI; ++j) {
            const long long row = wr0 + j * 16 + fl;
#pragma unroll
            for (int i = 0; i < QI; ++i) {
                const long long c = wc0 + i * 16 + fk * 4;
                if (row >= live || c >= p.cols) continue;        // (out_ld is a multiple of 4)
                f32x4* o = reinterpret_cast<f32x4*>(out + row * p.out_ld + c);
                f32x4 x = acc[i][j];
                if (p.add) x += *o;
                *o = x;
            }
        }
    } else {
        const float f = p.scale ? *p.scale : 1.f;
#pragma unroll
        for (int j = 0; j < RI; ++j) {
            const long long row = wr0 + j * 16 + fl;
#pragma unroll
            for (int i = 0; i < QI; ++i) {
                const long long c = wc0 + i * 16 + fk * 4;
                if (row >= p.r_rows || c >= p.cols) continue;
                const f32x4 x = acc[i][j] * f;
                if (p.out_bf16) {
                    bf16_t* o = static_cast<bf16_t*>(p.out) + row * p.out_ld + c;
                    if ((p.out_ld & 3) == 0) {
                        bf16x4 q;
                        for (int e = 0; e < 4; ++e) q[e] = (bf16_t)x[e];
                        *reinterpret_cast<bf16x4*>(o) = q;
                    } else {
                        for (int e = 0; e < 4; ++e)
                            if (c + e < p.cols) o[e] = (bf16_t)x[e];
                    }
                } else {
                    float* o = static_cast<float*>(p.out) + row * p.out_ld + c;
                    for (int e = 0; e < 4; ++e)
                        if (c + e < p.cols) o[e] = p.add ? o[e] + x[e] : x[e];
                }
            }
        }
    }
}

// ---- joins -------------------------------------------------------------------------------------------------------------------
// A lane per row, sixteen wavefronts over the tiles.
__global__ __launch_bounds__(1024) void join_stats_k(const float2* __restrict__ part, long long part_ld, int tiles, State s,
                                                     const float* __restrict__ target_logit, int reduction, float* __restrict__ loss,
                                                     float* __restrict__ row_loss) {
    __shared__ float2 sm[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, count = *s.count;
    const int row = blockIdx.x * 64 + lane;
    if ((int)(blockIdx.x * 64) >= count) return;
    float m = -INFINITY, sum = 0.f;
    for (int t = wave; t < tiles; t += 16) {
        const float2 q = part[t * part_ld + row];
        const float n = q.x > m ? q.x : m, ns = n == -INFINITY ? 0.f : n;
        sum = sum * expf(m - ns) + q.y * expf(q.x - ns);
        m = n;
    }
    sm[wave][lane] = make_float2(m, sum);
    __syncthreads();
    if (wave != 0 || row >= count) return;
    for (int w = 1; w < 16; ++w) {
        const float2 q = sm[w][lane];
        const float n = q.x > m ? q.x : m, ns = n == -INFINITY ? 0.f : n;
        sum = sum * expf(m - ns) + q.y * expf(q.x - ns);
        m = n;
    }
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

// factor[0]: of all rows (mean, sum), or factor[r]: of each packed row
__global__ __launch_bounds__(256) void factors_k(const float* __restrict__ grad_out, State s, int reduction, float* __restrict__ factor) {
    const int n = *s.count;
    if (reduction != S2AG_LCE_NONE) {
        if (blockIdx.x == 0 && threadIdx.x == 0) *factor = reduction == S2AG_LCE_MEAN ? *grad_out / (float)(n > 0 ? n : 1) : *grad_out;
        return;
    }
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) factor[i] = grad_out[s.rowmap[i]];
}

// dx[r] = factor * sum over the splits of the packed row, zeros for rows that were ignored
template <typename T>
__global__ __launch_bounds__(256) void finish_dx_k(const float* __restrict__ acc, long long ld, long long split, int splits, State s,
                                                   const float* __restrict__ scale, long long rows, int dim, T* __restrict__ dx) {
    const float f = scale ? *scale : 1.f;
    const int groups = (dim + 3) / 4;
    const long long total = rows * groups;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / groups;
        const int c = (int)(i - r * groups) * 4, at = s.inv[r];
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        if (at >= 0) {
            for (int k = 0; k < splits; ++k) x += *reinterpret_cast<const f32x4*>(acc + k * split + at * ld + c);
            x *= f;
        }
        T* o = dx + r * dim + c;
        for (int e = 0; e < 4; ++e)
            if (c + e < dim) o[e] = (T)x[e];
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------
struct Plan {
    int planes, pairs;
    long long np, vp;                   // rows and words, padded
    int kp;
    bool pack_w;
    // bytes from the workspace's start
    long long xp, wp, part, tl, row_loss, xt, wt, factor, acc, g, gt, bytes;
    long long piece;                    // words of a piece of the vocabulary
    int splits, acc_ld;
};

constexpr long long PIECE_VALUES = 1LL << 27;   // of G in a piece: 256 MB each way in bf16, beside which the fp32 sums of dX are small

bool valid(const s2ag_lce_args* a) {
    // 2^21: a tile's rows stay within a 31-bit byte offset whichever way they run
    return a && a->rows >= 0 && a->rows <= (1 << 21) && a->vocab > 0 && a->vocab <= (1 << 21) && a->dim > 0 && a->dim <= (1 << 20) &&
           a->ldx >= a->dim && a->ldw >= a->dim && a->reduction >= 0 && a->reduction <= 2 && !(a->bf16 && a->dw_accumulate);
}

// 256 x 256 tiles where they fill the 256 compute units, else 128 x 128
bool big_tiles(long long r, long long q) { return cdiv(r, 256) * (long long)cdiv(q, 256) >= 256; }

Plan plan(const s2ag_lce_args* a, bool backward) {
    Plan p{};
    p.planes = a->bf16 ? 1 : 3;
    p.pairs = a->bf16 ? 1 : 6;
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
    p.xp = take(2 * p.planes * p.np * p.kp);
    p.wp = take(p.pack_w ? 2 * p.planes * a->vocab * p.kp : 0);
    if (!backward) {
        p.part = take(8 * p.np * cdiv(a->vocab, 128));
        p.tl = take(4 * p.np);
        p.row_loss = take(4 * p.np);
    } else {
        const long long most = PIECE_VALUES / p.planes / (p.np ? p.np : 1) / 256 * 256;
        const long long pieces = cdiv(p.vp, most < 1024 ? 1024 : most);
        p.piece = round_up(cdiv(p.vp, pieces), 256);
        const bool dx = a->dx != nullptr, dw = a->dw != nullptr;
        p.acc_ld = (int)round_up(a->dim, 4);
        // few tiles: the words of a piece are split, down to 16 stages each
        const bool big = big_tiles(p.np, a->dim);
        const long long tiles = (long long)cdiv(p.np, big ? 256 : 128) * cdiv(a->dim, big ? 256 : 128);
        long long s = cdiv(512, tiles ? tiles : 1);
        const long long stages = p.piece / BK * p.pairs;
        if (s > stages / 16) s = stages / 16;
        p.splits = big || s < 1 ? 1 : (int)s;
        p.xt = take(dw ? 2 * p.planes * a->dim * p.np : 0);
        p.wt = take(dx ? 2 * p.planes * a->dim * p.vp : 0);
        p.factor = take(4 * (a->reduction == S2AG_LCE_NONE ? p.np : 1));
        p.acc = take(dx ? 4 * p.splits * p.np * p.acc_ld : 0);
        p.g = take(dx ? 2 * p.planes * p.np * p.piece : 0);
        p.gt = take(dw ? 2 * p.planes * p.np * p.piece : 0);
    }
    p.bytes = at;
    return p;
}

template <int BR, int BQ, int WR, int WQ, End END>
int launch_tiles(Product& p, long long r_rows, long long q_rows, hipStream_t st) {
    constexpr int LDS = 2 * (BR + BQ) * BK * 2;
    static_assert(LDS >= BR * BQ * 2 && LDS >= WQ * BR * 8, "the ends reuse the stages");
    // (every time: the attribute belongs to the current device)
    if (hipFuncSetAttribute((const void*)product_k<BR, BQ, WR, WQ, END>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
        return S2AG_E_UNSUPPORTED;
    p.tiles_r = cdiv(r_rows, BR);
    p.tiles_q = cdiv(q_rows, BQ);
    const long long n = (long long)p.tiles_r * p.tiles_q * p.splits;
    if (n > 0x7fffffffLL) return S2AG_E_UNSUPPORTED;
    if (n == 0) return 0;
    hipLaunchKernelGGL((product_k<BR, BQ, WR, WQ, END>), dim3((unsigned)n), dim3(64 * WR * WQ), LDS, st, p);
    S2AG_LAUNCH_CHECK();
    return 0;
}

template <End END>
int launch(Product& p, long long r_rows, long long q_rows, hipStream_t st) {
    if (p.splits < 1) p.splits = 1;
    return big_tiles(r_rows, q_rows) ? launch_tiles<256, 256, 2, 2, END>(p, r_rows, q_rows, st)
                                     : launch_tiles<128, 128, 2, 2, END>(p, r_rows, q_rows, st);
}

unsigned grid_of(long long work) {
    const long long b = (work + 255) / 256;
    return (unsigned)(b < 1 ? 1 : b > 4096 ? 4096 : b);
}

int pack(const s2ag_lce_args* a, const Plan& p, const State& s, char* ws, Operand* x, Operand* w, hipStream_t st) {
    bf16_t* xp = reinterpret_cast<bf16_t*>(ws + p.xp);
    *x = Operand{xp, p.np * p.kp, p.kp};
    const unsigned g = grid_of(p.np * (p.kp / 8));
    if (a->bf16)
        hipLaunchKernelGGL(pack_k<bf16_t>, dim3(g), dim3(256), 0, st, static_cast<const bf16_t*>(a->x), a->ldx, a->dim, s.rowmap, s.count,
                           p.np, xp, p.kp, p.np * p.kp);
    else
        hipLaunchKernelGGL(pack_k<float>, dim3(g), dim3(256), 0, st, static_cast<const float*>(a->x), a->ldx, a->dim, s.rowmap, s.count, p.np,
                           xp, p.kp, p.np * p.kp);
    S2AG_LAUNCH_CHECK();
    if (!p.pack_w) {
        *w = Operand{static_cast<const bf16_t*>(a->w), 0, a->ldw};
        return 0;
    }
    bf16_t* wp = reinterpret_cast<bf16_t*>(ws + p.wp);
    *w = Operand{wp, a->vocab * p.kp, p.kp};
    const unsigned gw = grid_of(a->vocab * (p.kp / 8));
    if (a->bf16)
        hipLaunchKernelGGL(pack_k<bf16_t>, dim3(gw), dim3(256), 0, st, static_cast<const bf16_t*>(a->w), a->ldw, a->dim, (const int*)nullptr,
                           (const int*)nullptr, a->vocab, wp, p.kp, a->vocab * p.kp);
    else
        hipLaunchKernelGGL(pack_k<float>, dim3(gw), dim3(256), 0, st, static_cast<const float*>(a->w), a->ldw, a->dim, (const int*)nullptr,
                           (const int*)nullptr, a->vocab, wp, p.kp, a->vocab * p.kp);
    S2AG_LAUNCH_CHECK();
    return 0;
}

bool ready(const s2ag_lce_args* a, const Plan& p) {
    return a->x && a->w && a->target && a->state && a->workspace && a->workspace_bytes >= p.bytes && aligned16(a->workspace) && aligned16(a->state);
}
}  // namespace

extern "C" long long s2ag_lce_state_bytes(long long rows) {
    if (rows < 0 || rows > (1 << 21)) return S2AG_E_BADARG;
    return 4 * state_words(rows);
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
    hipLaunchKernelGGL(select_rows_k, dim3(1), dim3(1024), 0, st, a->target, a->target_i32, a->rows, a->vocab, a->ignore_index, s,
                       a->reduction == S2AG_LCE_NONE ? a->loss : nullptr);
    S2AG_LAUNCH_CHECK();
    if (a->rows) {
        Product q{};
        if (int rc = pack(a, p, s, ws, &q.r, &q.q, st)) return rc;
        q.r_rows = p.np;
        q.q_rows = q.vocab = a->vocab;
        q.k = p.kp;
        q.pairs = p.pairs;
        q.r_count = s.count;
        q.tgt = s.tgt;
        q.part = reinterpret_cast<float2*>(ws + p.part);
        q.part_ld = p.np;
        q.target_logit = reinterpret_cast<float*>(ws + p.tl);
        if (int rc = launch<STATS>(q, p.np, a->vocab, st)) return rc;
        hipLaunchKernelGGL(join_stats_k, dim3((unsigned)(p.np / 64)), dim3(1024), 0, st, q.part, q.part_ld, q.tiles_q, s, q.target_logit,
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
    float* factor = reinterpret_cast<float*>(ws + p.factor);
    const bool each = a->reduction == S2AG_LCE_NONE;
    hipLaunchKernelGGL(factors_k, dim3(each ? grid_of(a->rows) : 1), dim3(256), 0, st, a->grad_out, s, a->reduction, factor);
    S2AG_LAUNCH_CHECK();
    Operand x, w;
    if (int rc = pack(a, p, s, ws, &x, &w, st)) return rc;
    bf16_t* xt = reinterpret_cast<bf16_t*>(ws + p.xt);
    bf16_t* wt = reinterpret_cast<bf16_t*>(ws + p.wt);
    if (a->dw && p.np) {
        hipLaunchKernelGGL(transpose_k, dim3((unsigned)(p.np / 64), cdiv(a->dim, 64), p.planes), dim3(256), 0, st, x, p.np, s.count, a->dim, xt,
                           p.np, a->dim * p.np);
        S2AG_LAUNCH_CHECK();
    }
    if (a->dx && p.np) {
        hipLaunchKernelGGL(transpose_k, dim3((unsigned)(p.vp / 64), cdiv(a->dim, 64), p.planes), dim3(256), 0, st, w, a->vocab,
                           (const int*)nullptr, a->dim, wt, p.vp, a->dim * p.vp);
        S2AG_LAUNCH_CHECK();
    }
    bf16_t* g = reinterpret_cast<bf16_t*>(ws + p.g);
    bf16_t* gt = reinterpret_cast<bf16_t*>(ws + p.gt);
    float* acc = reinterpret_cast<float*>(ws + p.acc);
    for (long long v0 = 0; v0 < p.vp; v0 += p.piece) {
        const long long words = a->vocab - v0 < p.piece ? a->vocab - v0 : p.piece;     // that exist
        if (words <= 0) break;
        const long long wide = round_up(words, 256);
        Product q{};
        q.r = x;
        q.q = Operand{w.p + v0 * w.ld, w.plane, w.ld};
        q.r_rows = p.np;
        q.q_rows = words;
        q.k = p.kp;
        q.pairs = p.pairs;
        q.r_count = s.count;
        q.tgt = s.tgt;
        q.q0 = v0;
        q.vocab = a->vocab;
        q.lse = s.lse;
        q.factor = each ? factor : nullptr;
        q.g = a->dx ? g : nullptr;
        q.g_ld = p.piece;
        q.g_plane = p.np * p.piece;
        q.gt = a->dw ? gt : nullptr;
        q.gt_ld = p.np;
        q.gt_plane = p.piece * p.np;
        if (int rc = launch<GRADS>(q, p.np, wide, st)) return rc;
        if (a->dx) {
            Product d{};
            d.r = Operand{g, q.g_plane, p.piece};
            d.q = Operand{wt + v0, a->dim * p.vp, p.vp};
            d.r_rows = p.np;
            d.q_rows = d.cols = a->dim;
            d.k = (int)wide;
            d.pairs = p.pairs;
            d.r_count = s.count;
            d.splits = p.splits;
            d.out = acc;
            d.out_ld = p.acc_ld;
            d.out_split = p.np * p.acc_ld;
            d.add = v0 > 0;
            if (int rc = launch<ACCUM>(d, p.np, a->dim, st)) return rc;
        }
        if (a->dw) {
            Product d{};
            d.r = Operand{gt, q.gt_plane, p.np};
            d.q = Operand{xt, a->dim * p.np, p.np};
            d.r_rows = words;
            d.q_rows = d.cols = a->dim;
            d.k_count = s.count;
            d.pairs = p.pairs;
            d.out = a->bf16 ? (void*)(static_cast<bf16_t*>(a->dw) + v0 * a->dim) : (void*)(static_cast<float*>(a->dw) + v0 * a->dim);
            d.out_ld = a->dim;
            d.out_bf16 = a->bf16;
            d.add = a->dw_accumulate;
            d.scale = each ? nullptr : factor;
            if (int rc = launch<STORE>(d, words, a->dim, st)) return rc;
        }
    }
    if (a->dx && a->rows) {
        const unsigned gx = grid_of(a->rows * ((a->dim + 3) / 4));
        if (a->bf16)
            hipLaunchKernelGGL(finish_dx_k<bf16_t>, dim3(gx), dim3(256), 0, st, acc, (long long)p.acc_ld, p.np * p.acc_ld, p.splits, s,
                               each ? nullptr : factor, a->rows, a->dim, static_cast<bf16_t*>(a->dx));
        else
            hipLaunchKernelGGL(finish_dx_k<float>, dim3(gx), dim3(256), 0, st, acc, (long long)p.acc_ld, p.np * p.acc_ld, p.splits, s,
                               each ? nullptr : factor, a->rows, a->dim, static_cast<float*>(a->dx));
        S2AG_LAUNCH_CHECK();
    }
    return 0;
}
