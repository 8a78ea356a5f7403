// ssla_linattn_chunk.cu -- linear attention over whole sequences, 64 tokens
// (a chunk) at a time on the tensor cores.
//
// With G_t the sum of a chunk's log decays up to token t and S_0 the state
// before the chunk,
//     out_t = scale (e^{G_t} q_t S_0 + sum_{s<=t} e^{G_t - G_s} (q_t . k_s) v_s)
//     S     = e^{G_C} S_0 + sum_s e^{G_C - G_s} k_s v_s^T
// so that a chunk is four small matrix products and the state moves once per
// chunk.  A CTA walks the chunks of one segment of a sequence for one head
// and DV state columns, the state in registers.
//
// Precision.  The matrix instructions take bf16 operands and add in 32 bits.
// A 32-bit operand goes through as the sum of bf16 pieces (8 bits each):
// bf16 inputs are one piece and exact, fp16 two and exact, fp32 three.
// What is computed (decayed scores, decayed keys, the state) goes through as
// two pieces, 2^-16, where it only reaches a 16-bit output, as three, 2^-24,
// where it reaches a 32-bit output or the state.  Products of pieces whose
// combined order is below those are left out.  Each chunk's sum is added to
// the state by an ordinary 32-bit fma, so that the truncating adders of the
// matrix unit never accumulate over a sequence.
//
// Long sequences.  Where the sequences and heads alone do not fill the GPU, a
// sequence is divided into segments: k_chunk<OUT = false> leaves every
// segment's own end state (from zero) and decay in the workspace,
// k_chunk_join chains them into the segments' first states, and
// k_chunk<OUT = true> runs all segments at once.
//
// Measured: 8 sequences of 25,000 tokens, 4 heads of 24, fp32: 340 us, bound by
// issue slots (8,265 warp instructions a chunk and head, 3,960 in the pass for
// the segments' own states); the products themselves are a fifth of that.
//
// Non-finite values.  A value in token s may not reach the outputs of tokens
// before s, but 0 * inf in a masked place would take it there.  Masked scores
// are replaced, not multiplied, and a non-finite v is taken out of the tile
// and put back as NaN into its column from its own token on.
//
// Clears.  A decay of -infinity replaces the state by zero, whatever it holds.
// As a decay of -1e5 it takes every finite value before it to zero in the
// products above; 0 * infinity would stay, in the state too.  So a CTA that
// ends with a state that is not finite looks for a clear among its decays, and
// where there is one goes through its tokens again, one by one (walk): 0.7 us a
// token, 3.5 us in the tcgen05 form.  The others pay 1 to 3 % for the question.
// Masks for the tokens from one clear to the next, in the products themselves,
// cost every call 2 to 20 %.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "ssla_linattn.cuh"

namespace ssla {
namespace ops {
namespace {

constexpr int kChunk = 64;
constexpr int kThreads = 128;
constexpr int kTable = 256;          // sequences of one launch

struct Table {
    int n;
    int start[kTable], len[kTable], slot[kTable];
    int seg0[kTable + 1];            // first segment of each sequence
    int step[kTable];                // tokens of a segment (a multiple of kChunk)
};

// Pieces of the inputs and of what reaches only the outputs.
template <typename T> struct Pieces;
template <> struct Pieces<float> { static constexpr int in = 3, mid = 3, order = 2; };
template <> struct Pieces<__half> { static constexpr int in = 2, mid = 2, order = 1; };
template <> struct Pieces<__nv_bfloat16> { static constexpr int in = 1, mid = 2, order = 1; };

template <typename T, int DK, int DV> struct Tile {
    static constexpr int IN = Pieces<T>::in, MID = Pieces<T>::mid;
    static constexpr int LK = DK + 8, LV = DV + 8;      // row lengths: 16-byte rows on distinct banks
    static constexpr int kQ = 0, kK = kQ + IN * kChunk * LK, kV = kK + IN * kChunk * LK,
                         kS = kV + IN * kChunk * LV, kEnd = kS + MID * DK * LV;
    static constexpr int bytes = kEnd * 2 + (4 * kChunk + 4 + DV) * 4;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const __nv_bfloat16* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_addr(p)));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const __nv_bfloat16* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_addr(p)));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c0, c1 += the product of a (NA pieces) and b (NB pieces, columns of two
// tiles), pieces of combined order up to ORD, the smallest first.  The matrix
// unit's adder truncates; FRESH (32-bit results) lets it add only one step's
// products and rounds the step into c.
template <int ORD, bool FRESH, int NA, int NB>
__device__ __forceinline__ void mma_pieces(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][4]) {
    float t0[4] = {}, t1[4] = {};
#pragma unroll
    for (int o = ORD; o >= 0; --o)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (o - i >= 0 && o - i < NB) {
                mma(FRESH ? t0 : c0, a[i], b[o - i][0], b[o - i][1]);
                mma(FRESH ? t1 : c1, a[i], b[o - i][2], b[o - i][3]);
            }
    if (FRESH)
#pragma unroll
        for (int e = 0; e < 4; ++e) c0[e] += t0[e], c1[e] += t1[e];
}

__device__ __forceinline__ uint32_t pack2(float x, float y) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ float2 unpack2(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
// The first of several pieces: 32-bit values above bf16's largest give that,
// not infinity, and leave the rest to the next piece; so do infinities, whose
// next piece is one.
__device__ __forceinline__ uint32_t pack2_finite(float x, float y) {
    uint32_t p;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(y), "f"(x));
    return p;
}
// The next piece of (x, y); what is left stays in them.
template <bool FIRST = false> __device__ __forceinline__ uint32_t take(float& x, float& y) {
    const uint32_t p = FIRST ? pack2_finite(x, y) : pack2(x, y);
    const float2 f = unpack2(p);
    x -= f.x;
    y -= f.y;
    return p;
}
__device__ __forceinline__ float exp2_fast(float x) {     // 2^-22; results below 2^-126 become zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// Eight values of a row at p + c (zero from `width` on).
template <typename T>
__device__ __forceinline__ void load8(const T* p, int c, int width, bool wide, float (&x)[8]) {
    if (wide && c + 8 <= width) {
        if constexpr (sizeof(T) == 2) {
            load_vec<T, 8>(p + c, x);
        } else {
            float lo[4], hi[4];
            load_vec<T, 4>(p + c, lo);
            load_vec<T, 4>(p + c + 4, hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = lo[j], x[j + 4] = hi[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = c + j < width ? to_f<T>(p[c + j]) : 0.0f;
    }
}

// Rows [0, rows) x [0, width) of a token tile, on the way from global memory:
// thread t's eight values of row (t + i * kThreads) / (D / 8).
template <int D> struct Moving {
    static constexpr int N = kChunk * (D / 8) / kThreads;
    float x[N][8];

    template <typename T> __device__ void load(const T* p, long long stride, int rows, int width, bool wide) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = threadIdx.x + i * kThreads, r = e / (D / 8), c = e % (D / 8) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = 0.0f;
            if (r < rows && c < width) load8<T>(p + r * stride, c, width, wide, x[i]);
        }
    }
    // To shared memory as IN pieces.  With `bad`, non-finite values become
    // zero and their first row is noted by column.
    template <int IN> __device__ bool store(__nv_bfloat16* s, int* bad) {
        constexpr int LD = D + 8;
        bool any = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = threadIdx.x + i * kThreads, r = e / (D / 8), c = e % (D / 8) * 8;
            if (bad) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!finite(x[i][j])) {
                        atomicMin(bad + c + j, r);
                        x[i][j] = 0.0f;
                        any = true;
                    }
            }
#pragma unroll
            for (int n = 0; n < IN; ++n) {
                uint4 u;
                if (IN == 3 && n == 0) {           // (16-bit inputs are not above bf16's largest)
                    u.x = take<true>(x[i][0], x[i][1]); u.y = take<true>(x[i][2], x[i][3]);
                    u.z = take<true>(x[i][4], x[i][5]); u.w = take<true>(x[i][6], x[i][7]);
                } else {
                    u.x = take(x[i][0], x[i][1]); u.y = take(x[i][2], x[i][3]);
                    u.z = take(x[i][4], x[i][5]); u.w = take(x[i][6], x[i][7]);
                }
                *reinterpret_cast<uint4*>(s + n * kChunk * LD + r * LD + c) = u;
            }
        }
        return any;
    }
};

// Asks for the lines of rows [0, rows) x `bytes` in L2.
template <typename T> __device__ __forceinline__ void fetch_ahead(const T* p, long long stride, int rows, int width) {
    for (int r = threadIdx.x; r < rows; r += kThreads)
        for (int c = 0; c < width; c += 128 / static_cast<int>(sizeof(T)))
            asm volatile("prefetch.global.L2 [%0];" ::"l"(p + r * stride + c));
}

// One float2 of a state row, bounds-checked.
__device__ __forceinline__ float2 state_load2(const float* p, int r, int c, int dk, int dv) {
    float2 x = make_float2(0.0f, 0.0f);
    if (r < dk) {
        if (c < dv) x.x = p[static_cast<size_t>(r) * dv + c];
        if (c + 1 < dv) x.y = p[static_cast<size_t>(r) * dv + c + 1];
    }
    return x;
}
__device__ __forceinline__ void state_store2(float* p, int r, int c, int dk, int dv, float x, float y) {
    if (r < dk) {
        if (c < dv) p[static_cast<size_t>(r) * dv + c] = x;
        if (c + 1 < dv) p[static_cast<size_t>(r) * dv + c + 1] = y;
    }
}

// The log decays of tokens 2 lane and 2 lane + 1 of a chunk (0 from token n on).
__device__ __forceinline__ float2 chunk_decay_values(const LinArgs& a, long long row, int n, int h, int lane) {
    const float* p = a.decay + row * a.decay_row + h * a.decay_head;
    const int t = 2 * lane;
    return make_float2(t < n ? p[t * a.decay_row] : 0.0f, t + 1 < n ? p[(t + 1) * a.decay_row] : 0.0f);
}

// A chunk's decay sums, by one warp; a lane's for its two tokens: G_t = sum of
// the log2 decays up to token t as (hi, lo), 2^{G_t}, 2^{G_C - G_t}, and for
// the chunk 2^{G_C} and G_C.  The sums are taken in 64 bits: differences of
// them are exponents.
struct DecaySums {
    float hi[2], lo[2], grown[2], left[2], whole;
    double total;
};
__device__ __forceinline__ DecaySums chunk_decays(float2 g, int lane) {
    DecaySums d;
    double s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float x = j ? g.y : g.x;
        if (x < -1e5f) x = -1e5f;                           // e^-1e5 is 0 as well, and -inf - -inf is not
        s[j] = x * 1.4426950408889634;
    }
    s[1] += s[0];
    double run = s[1];
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const double o = __shfl_up_sync(0xFFFFFFFFu, run, m);
        if (lane >= m) run += o;
    }
    d.total = __shfl_sync(0xFFFFFFFFu, run, 31);
    double before = __shfl_up_sync(0xFFFFFFFFu, run, 1);    // (not run - s[1]: a NaN there is this lane's second token's)
    if (lane == 0) before = 0.0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const double G = j ? run : before + s[0];
        d.hi[j] = static_cast<float>(G);
        d.lo[j] = static_cast<float>(G - d.hi[j]);
        d.grown[j] = exp2f(d.hi[j]);
        d.left[j] = exp2f(static_cast<float>(d.total - G));
    }
    d.whole = exp2f(static_cast<float>(d.total));
    return d;
}

// The recurrence itself, over rows [row0, row0 + count) of head h, by
// THREADS = COLS * PARTS threads (`tid`, which meet at sync()): thread (col,
// part) has state rows [part * N, part * N + N) of value column c0 + col, from
// `from` (null: zero) to `to` (null: nowhere).  mem: walk_floats of shared
// memory.  A token's keys and queries pass through it, the next token's in
// flight; with SHARED the state is there as well (where registers are short).
// Returns the sum of the log2 decays, -infinity with a clear.
template <int DK, int COLS, int PARTS, bool SHARED> constexpr int walk_floats = 4 * DK + 2 * COLS * PARTS + (SHARED ? DK * COLS : 0);
template <typename T, int DK, int COLS, int PARTS, bool OUT, bool SHARED, typename Sync>
__device__ __forceinline__ double walk(const LinArgs& a, int h, long long row0, int count, int c0, int tid, const float* from, float* to, float* mem,
                                       Sync sync) {
    constexpr int N = DK / PARTS, THREADS = COLS * PARTS, MOVES = (2 * DK + THREADS - 1) / THREADS;
    const int col = c0 + tid % COLS, part = tid / COLS, k0 = part * N;
    const bool live = col < a.dv;
    const int rows = live ? min(N, a.dk - k0) : 0;
    const T* q = static_cast<const T*>(a.q) + (h / a.q_share) * a.q_head + row0 * a.q_row;
    const T* k = static_cast<const T*>(a.k) + (h / a.k_share) * a.k_head + row0 * a.k_row;
    const T* v = static_cast<const T*>(a.v) + h * a.v_head + row0 * a.v_row + col;
    const float* decay = a.decay + h * a.decay_head + row0 * a.decay_row;
    T* out = static_cast<T*>(a.out) + h * a.out_head + row0 * a.out_row + col;
    float kept[SHARED ? 1 : N], move[MOVES], g = 0.0f, x = 0.0f;
    auto S = [&](int i) -> float& {
        if constexpr (SHARED) return mem[4 * DK + 2 * THREADS + i * THREADS + tid];
        else return kept[i];
    };
    constexpr int UNROLL = SHARED ? 8 : N;
#pragma unroll UNROLL
    for (int i = 0; i < N; ++i) S(i) = from && i < rows ? from[static_cast<size_t>(k0 + i) * a.dv + col] : 0.0f;
    auto ask = [&](int t) {
        g = decay[t * a.decay_row];
        x = live ? to_f<T>(v[t * a.v_row]) : 0.0f;
#pragma unroll
        for (int i = 0; i < MOVES; ++i) {
            const int e = tid + i * THREADS, c = e % DK;
            move[i] = e >= 2 * DK || c >= a.dk ? 0.0f : to_f<T>(e < DK ? k[t * a.k_row + c] : q[t * a.q_row + c]);
        }
    };
    ask(0);
    double total = 0.0;
#pragma unroll 1
    for (int t = 0; t < count; ++t) {
        float* const kq = mem + t % 2 * 2 * DK;
        float* const parts = mem + 4 * DK + t % 2 * THREADS;
#pragma unroll
        for (int i = 0; i < MOVES; ++i)
            if (tid + i * THREADS < 2 * DK) kq[tid + i * THREADS] = move[i];
        const float e = expf(g), vt = x;
        total = g == -INFINITY ? -INFINITY : total + g * 1.4426950408889634;
        if (g == -INFINITY)
#pragma unroll UNROLL
            for (int i = 0; i < N; ++i) S(i) = 0.0f;
        sync();
        if (t + 1 < count) ask(t + 1);
        float sums[4] = {};
#pragma unroll UNROLL
        for (int i = 0; i < N; ++i) {
            const float s = fmaf(kq[k0 + i], vt, e * S(i));
            S(i) = i < rows ? s : 0.0f;                     // (0 * NaN from dk on)
            sums[i % 4] = fmaf(kq[DK + k0 + i], i < rows ? s : 0.0f, sums[i % 4]);
        }
        if (OUT) {
            float o = (sums[0] + sums[1]) + (sums[2] + sums[3]);
            parts[tid] = o;
            sync();
            if (part == 0 && live) {
#pragma unroll
                for (int i = 1; i < PARTS; ++i) o += parts[tid + i * COLS];
                out[t * a.out_row] = from_f<T>(o * a.scale);
            }
        }
    }
    if (to)
#pragma unroll UNROLL
        for (int i = 0; i < N; ++i)
            if (i < rows) to[static_cast<size_t>(k0 + i) * a.dv + col] = S(i);
    return total;
}
// Whether one of the threads' decays (thread t of `threads`) is a clear.
__device__ __forceinline__ bool some_clear(const LinArgs& a, int h, long long row0, int count, int t, int threads) {
    bool found = false;
    for (; t < count; t += threads) found |= a.decay[(row0 + t) * a.decay_row + h * a.decay_head] == -INFINITY;
    return found;
}

// Segment states: [segment][head][dk][dv]; segment decays: [segment][head].
// Where a divided sequence's segment finds its first state: the place of the
// segment before it, the first one that of the last (which leaves none), since
// the slot itself may already hold the last segment's result.
__device__ __forceinline__ int first_state_of(const Table& tab, int seq, int seg) {
    return seg ? tab.seg0[seq] + seg - 1 : tab.seg0[seq + 1] - 1;
}

template <typename T, int DK, int DV, bool OUT>
__global__ void __launch_bounds__(kThreads, DK <= 32 && DV <= 32 ? 4 : 1)
k_chunk(LinArgs a, const __grid_constant__ Table tab, float* seg_state, double* seg_decay, int wide) {
    using L = Tile<T, DK, DV>;
    constexpr bool FRESH = sizeof(T) == 4;
    constexpr int IN = L::IN, MID = L::MID, ORD = Pieces<T>::order, LK = L::LK, LV = L::LV, NT = DV / 8;
    constexpr int MT = DK >= 64 ? DK / 64 : 1;            // 16-row state tiles of a warp
    constexpr int SN = DK >= 64 ? NT : NT / 2;            // and its 8-column tiles
    extern __shared__ __align__(16) uint8_t smem[];
    __nv_bfloat16* sb = reinterpret_cast<__nv_bfloat16*>(smem);
    __nv_bfloat16 *sQ = sb + L::kQ, *sK = sb + L::kK, *sV = sb + L::kV, *sS = sb + L::kS;
    float* ghi = reinterpret_cast<float*>(sb + L::kEnd);
    float *glo = ghi + kChunk, *wk = glo + kChunk, *eg = wk + kChunk, *gam = eg + kChunk;
    int* bad = reinterpret_cast<int*>(gam + 4);

    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g8 = lane / 4, t2 = lane % 4 * 2;
    const int h = blockIdx.y, c0 = blockIdx.x * DV;
    // this CTA's sequence and segment
    int lo = 0, hi = tab.n;
    while (hi - lo > 1) {
        const int m = (lo + hi) / 2;
        if (tab.seg0[m] <= static_cast<int>(blockIdx.z)) lo = m;
        else hi = m;
    }
    const int seq = lo, seg = blockIdx.z - tab.seg0[seq], nseg = tab.seg0[seq + 1] - tab.seg0[seq];
    if (!OUT && seg == nseg - 1) return;
    const int first = seg * tab.step[seq], last = first + min(tab.len[seq] - first, tab.step[seq]);
    const int slot = tab.slot[seq];
    const size_t head_state = static_cast<size_t>(a.dk) * a.dv;
    const int m0 = (DK >= 64 ? warp * MT : warp % 2) * 16, n0 = DK >= 64 ? 0 : warp / 2 * SN * 8;

    float S[MT][SN][4];
    const float* from = nullptr;
    if (OUT && nseg > 1) from = seg_state + (static_cast<size_t>(first_state_of(tab, seq, seg)) * a.heads + h) * head_state;
    else if (OUT && slot >= 0) from = a.state + (static_cast<size_t>(slot) * a.heads + h) * head_state;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < SN; ++j) {
            float2 x = make_float2(0.0f, 0.0f), y = x;
            if (from) {
                x = state_load2(from, m0 + i * 16 + g8, c0 + n0 + j * 8 + t2, a.dk, a.dv);
                y = state_load2(from, m0 + i * 16 + g8 + 8, c0 + n0 + j * 8 + t2, a.dk, a.dv);
            }
            S[i][j][0] = x.x; S[i][j][1] = x.y; S[i][j][2] = y.x; S[i][j][3] = y.y;
        }
    bool zero = from == nullptr;                           // S is zero: no product with it
    double total = 0.0;
    bool cleared = false;                                  // (this lane's tokens)

    const int row0 = tab.start[seq];
    const T* Q = static_cast<const T*>(a.q) + (h / a.q_share) * a.q_head;
    const T* K = static_cast<const T*>(a.k) + (h / a.k_share) * a.k_head;
    const T* V = static_cast<const T*>(a.v) + h * a.v_head + c0;

    if (tid < DV) bad[tid] = kChunk;
    __syncthreads();
    for (int c = first; c < last; c += kChunk) {
        const int n = min(kChunk, last - c);
        const long long row = static_cast<long long>(row0) + c;
        // ---- the chunk's tiles, decays and the state's pieces into shared memory ----
        bool any;
        {
            const T *q = Q + row * a.q_row, *k = K + row * a.k_row, *v = V + row * a.v_row;
            Moving<DV> mv;
            Moving<DK> mk;
            // all loads before the first store, where the registers are there
            mv.load(v, a.v_row, n, a.dv - c0, wide & 4);
            mk.load(k, a.k_row, n, a.dk, wide & 2);
            if constexpr (OUT && DK <= 32) {
                Moving<DK> mq;
                mq.load(q, a.q_row, n, a.dk, wide & 1);
                mq.template store<IN>(sQ, nullptr);
            }
            mk.template store<IN>(sK, nullptr);
            any = mv.template store<IN>(sV, bad);
            if constexpr (OUT && DK > 32) {
                Moving<DK> mq;
                mq.load(q, a.q_row, n, a.dk, wide & 1);
                mq.template store<IN>(sQ, nullptr);
            }
            const int ahead = min(kChunk, last - c - n);
            if (OUT) fetch_ahead(q + n * a.q_row, a.q_row, ahead, a.dk);
            fetch_ahead(k + n * a.k_row, a.k_row, ahead, a.dk);
            fetch_ahead(v + n * a.v_row, a.v_row, ahead, min(a.dv - c0, DV));
        }
        if (OUT && !zero) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < SN; ++j) {
                    float x0 = S[i][j][0], x1 = S[i][j][1], y0 = S[i][j][2], y1 = S[i][j][3];
                    __nv_bfloat16* p = sS + (m0 + i * 16 + g8) * LV + n0 + j * 8 + t2;
#pragma unroll
                    for (int m = 0; m < MID; ++m) {
                        *reinterpret_cast<uint32_t*>(p + m * DK * LV) = m ? take(x0, x1) : take<true>(x0, x1);
                        *reinterpret_cast<uint32_t*>(p + m * DK * LV + 8 * LV) = m ? take(y0, y1) : take<true>(y0, y1);
                    }
                }
        }
        if (warp == 0) {
            const float2 g = chunk_decay_values(a, row, n, h, lane);
            const DecaySums d = chunk_decays(g, lane);
            if (!OUT) cleared |= g.x == -INFINITY || g.y == -INFINITY;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int t = 2 * lane + j;
                ghi[t] = d.hi[j];
                glo[t] = d.lo[j];
                eg[t] = d.grown[j];
                wk[t] = d.left[j];
            }
            if (lane == 0) gam[0] = d.whole;
            total += d.total;
        }
        any = __syncthreads_or(any);

        if (OUT && warp * 16 < n) {
            const int r0 = warp * 16;
            float A[8][4], O[NT][4];
#pragma unroll
            for (int j = 0; j < 8; ++j) A[j][0] = A[j][1] = A[j][2] = A[j][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < NT; ++j) O[j][0] = O[j][1] = O[j][2] = O[j][3] = 0.0f;
            // ---- scores q k^T up to the diagonal, and q S ----
#pragma unroll 2
            for (int ks = 0; ks < DK; ks += 16) {
                if (ks >= a.dk) break;
                uint32_t qa[IN][4];
#pragma unroll
                for (int i = 0; i < IN; ++i)
                    ldsm4(qa[i], sQ + i * kChunk * LK + (r0 + lane % 16) * LK + ks + lane / 16 * 8);
#pragma unroll
                for (int p = 0; p < 4; ++p)
                    if (p <= warp) {
                        uint32_t b[IN][4];
#pragma unroll
                        for (int i = 0; i < IN; ++i)
                            ldsm4(b[i], sK + i * kChunk * LK + (p * 16 + lane % 8 + lane / 16 * 8) * LK + ks + lane / 8 % 2 * 8);
                        mma_pieces<IN == 1 ? 0 : ORD, FRESH>(A[2 * p], A[2 * p + 1], qa, b);
                    }
                if (!zero)
#pragma unroll
                    for (int p = 0; p < NT / 2; ++p) {
                        uint32_t b[MID][4];
#pragma unroll
                        for (int i = 0; i < MID; ++i)
                            ldsm4t(b[i], sS + i * DK * LV + (ks + lane % 16) * LV + p * 16 + lane / 16 * 8);
                        mma_pieces<ORD, FRESH>(O[2 * p], O[2 * p + 1], qa, b);
                    }
            }
            const int ra = r0 + g8, rb = ra + 8;
            const float ea = eg[ra], eb = eg[rb], ha = ghi[ra], la = glo[ra], hb = ghi[rb], lb = glo[rb];
#pragma unroll
            for (int j = 0; j < NT; ++j) O[j][0] *= ea, O[j][1] *= ea, O[j][2] *= eb, O[j][3] *= eb;
            // ---- decayed scores (masked ones replaced), times v ----
#pragma unroll
            for (int p = 0; p < 4; ++p)
                if (p <= warp && p * 16 < n) {
                    float P[2][4];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int s = p * 16 + j * 8 + t2 + e;
                            const float hs = ghi[s], ls = glo[s];
                            P[j][e] = s <= ra ? A[2 * p + j][e] * exp2_fast((ha - hs) + (la - ls)) : 0.0f;
                            P[j][2 + e] = s <= rb ? A[2 * p + j][2 + e] * exp2_fast((hb - hs) + (lb - ls)) : 0.0f;
                        }
                    uint32_t pa[MID][4];
#pragma unroll
                    for (int i = 0; i < MID; ++i) {
                        pa[i][0] = i ? take(P[0][0], P[0][1]) : take<true>(P[0][0], P[0][1]);
                        pa[i][1] = i ? take(P[0][2], P[0][3]) : take<true>(P[0][2], P[0][3]);
                        pa[i][2] = i ? take(P[1][0], P[1][1]) : take<true>(P[1][0], P[1][1]);
                        pa[i][3] = i ? take(P[1][2], P[1][3]) : take<true>(P[1][2], P[1][3]);
                    }
#pragma unroll
                    for (int m = 0; m < NT / 2; ++m) {
                        uint32_t b[IN][4];
#pragma unroll
                        for (int i = 0; i < IN; ++i)
                            ldsm4t(b[i], sV + i * kChunk * LV + (p * 16 + lane % 16) * LV + m * 16 + lane / 16 * 8);
                        mma_pieces<ORD, FRESH>(O[2 * m], O[2 * m + 1], pa, b);
                    }
                }
            if (any)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int b = bad[j * 8 + t2 + e];
                        if (ra >= b) O[j][e] = __int_as_float(0x7FC00000);
                        if (rb >= b) O[j][2 + e] = __int_as_float(0x7FC00000);
                    }
            T* po = static_cast<T*>(a.out) + h * a.out_head + c0;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int col = j * 8 + t2 + e;
                    if (c0 + col < a.dv) {
                        if (ra < n) po[(row + ra) * a.out_row + col] = from_f<T>(O[j][e] * a.scale);
                        if (rb < n) po[(row + rb) * a.out_row + col] = from_f<T>(O[j][2 + e] * a.scale);
                    }
                }
        }
        // ---- the state: decayed keys, transposed, times v ----
        const float gc = gam[0];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if (m0 + i * 16 >= a.dk) break;
            float U[SN][4];
#pragma unroll
            for (int j = 0; j < SN; ++j) U[j][0] = U[j][1] = U[j][2] = U[j][3] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < kChunk; ks += 16) {
                if (ks >= n) break;
                const int kr = ks + lane % 8 + lane / 16 * 8, kc = m0 + i * 16 + lane / 8 % 2 * 8;
                float2 f[4] = {};
#pragma unroll
                for (int m = IN - 1; m >= 0; --m) {         // the smallest first: the larger two may add up to above the largest float
                    uint32_t r[4];
                    ldsm4t(r, sK + m * kChunk * LK + kr * LK + kc);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 x = unpack2(r[e]);
                        f[e].x += x.x;
                        f[e].y += x.y;
                    }
                }
                const float w0 = wk[ks + t2], w1 = wk[ks + t2 + 1], w2 = wk[ks + t2 + 8], w3 = wk[ks + t2 + 9];
                f[0].x *= w0; f[0].y *= w1; f[1].x *= w0; f[1].y *= w1;
                f[2].x *= w2; f[2].y *= w3; f[3].x *= w2; f[3].y *= w3;
                uint32_t ka[3][4];
#pragma unroll
                for (int m = 0; m < 3; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) ka[m][e] = m ? take(f[e].x, f[e].y) : take<true>(f[e].x, f[e].y);
#pragma unroll
                for (int p = 0; p < SN / 2; ++p) {
                    uint32_t b[IN][4];
#pragma unroll
                    for (int m = 0; m < IN; ++m)
                        ldsm4t(b[m], sV + m * kChunk * LV + (ks + lane % 16) * LV + n0 + p * 16 + lane / 16 * 8);
                    mma_pieces<2, FRESH>(U[2 * p], U[2 * p + 1], ka, b);
                }
            }
#pragma unroll
            for (int j = 0; j < SN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    S[i][j][e] = fmaf(gc, S[i][j][e], U[j][e]);
                    if (any && bad[n0 + j * 8 + t2 + e % 2] < kChunk) S[i][j][e] = __int_as_float(0x7FC00000);
                }
        }
        zero = false;
        __syncthreads();                                    // the tiles are rewritten
        if (any) {
            if (tid < DV) bad[tid] = kChunk;
            __syncthreads();
        }
    }

    float* to = nullptr;
    if (!OUT) to = seg_state + (static_cast<size_t>(blockIdx.z) * a.heads + h) * head_state;
    else if (seg == nseg - 1 && slot >= 0 && last > first)
        to = a.state + (static_cast<size_t>(slot) * a.heads + h) * head_state;
    if (!OUT && warp == 0 && __any_sync(0xFFFFFFFFu, cleared)) total = -INFINITY;
    float nought[4] = {};                                  // NaN where one is not finite
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < SN; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) nought[e] = fmaf(S[i][j][e], 0.0f, nought[e]);
    const bool fine = (nought[0] + nought[1]) + (nought[2] + nought[3]) == 0.0f;
    const long long row1 = static_cast<long long>(row0) + first;
    if (__syncthreads_or(!fine) && __syncthreads_or(some_clear(a, h, row1, last - first, tid, kThreads))) {
        static_assert(walk_floats<DK, DV, kThreads / DV, false> * 4 <= L::bytes, "shared memory");
        total = walk<T, DK, DV, kThreads / DV, OUT, false>(a, h, row1, last - first, c0, tid, from, to, reinterpret_cast<float*>(smem),
                                                    [] { __syncthreads(); });
        to = nullptr;
    }
    if (to)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < SN; ++j) {
                const int r = m0 + i * 16 + g8, c = c0 + n0 + j * 8 + t2;
                state_store2(to, r, c, a.dk, a.dv, S[i][j][0], S[i][j][1]);
                state_store2(to, r + 8, c, a.dk, a.dv, S[i][j][2], S[i][j][3]);
            }
    if (!OUT && blockIdx.x == 0 && tid == 0) seg_decay[static_cast<size_t>(blockIdx.z) * a.heads + h] = total;
}

#include "ssla_linattn_tc.cuh"

// Chains a sequence's segments: segment i's place in the workspace becomes
// the state after it, the last one's the state before all.  One thread per
// state element.
__global__ void __launch_bounds__(256)
k_chunk_join(LinArgs a, const __grid_constant__ Table tab, float* seg_state, const double* seg_decay) {
    const int seq = blockIdx.z, h = blockIdx.y;
    const int s0 = tab.seg0[seq], s1 = tab.seg0[seq + 1] - 1;
    const int e = blockIdx.x * 256 + threadIdx.x;
    if (s0 >= s1 || e >= a.dk * a.dv) return;
    const size_t head_state = static_cast<size_t>(a.dk) * a.dv;
    const int slot = tab.slot[seq];
    float run = slot >= 0 ? a.state[(static_cast<size_t>(slot) * a.heads + h) * head_state + e] : 0.0f;
    seg_state[(static_cast<size_t>(s1) * a.heads + h) * head_state + e] = run;
    for (int s = s0; s < s1; s += 8) {
        float x[8], g[8];                                   // loads of eight segments in flight
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (s + i < s1) {
                x[i] = seg_state[(static_cast<size_t>(s + i) * a.heads + h) * head_state + e];
                const double d = seg_decay[static_cast<size_t>(s + i) * a.heads + h];
                g[i] = d == -INFINITY ? -1.0f : exp2f(static_cast<float>(d));   // negative: a clear
            }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (s + i < s1) {
                run = g[i] < 0.0f ? x[i] : fmaf(g[i], run, x[i]);
                seg_state[(static_cast<size_t>(s + i) * a.heads + h) * head_state + e] = run;
            }
    }
}

// ---- host ------------------------------------------------------------------
struct Shape {
    int dk, dv, ctas;               // tile and resident CTAs per SM
    bool tc;                        // the tcgen05 form
    int cost;                       // a divided sequence's time over a whole one's, percent
    double setup, launches;         // in chunks' times: a segment's set-up and state traffic; the two further launches
};

template <typename F> auto with_shape(int dtype, int dk, int dv, F&& f) {
    auto by_dk = [&](auto t, auto v) {
        using std::integral_constant;
        if (dk <= 32) return f(t, integral_constant<int, 32>(), v);
        if (dk <= 64) return f(t, integral_constant<int, 64>(), v);
        return f(t, integral_constant<int, 128>(), v);
    };
    auto by_dv = [&](auto t) {
        return dv <= 32 ? by_dk(t, std::integral_constant<int, 32>()) : by_dk(t, std::integral_constant<int, 64>());
    };
    return dtype == SSLA_DT_F32 ? by_dv(float()) : dtype == SSLA_DT_BF16 ? by_dv(__nv_bfloat16()) : by_dv(__half());
}

// Which inputs allow 16-byte loads: bits 1 q, 2 k, 4 v.
int wide_inputs(const LinArgs& a, int dtype) {
    const int lanes = 16 / dtype_size(dtype);
    auto wide = [&](const void* p, long long row, long long head) {
        return aligned(p, 16) && row % lanes == 0 && head % lanes == 0;
    };
    return (wide(a.q, a.q_row, a.q_head) ? 1 : 0) | (wide(a.k, a.k_row, a.k_head) ? 2 : 0) |
           (wide(a.v, a.v_row, a.v_head) ? 4 : 0);
}

Shape shape_of(const LinArgs& a, int dtype) {
    // bf16 with wide heads: the tcgen05 form, whose copies are 16 bytes wide
    if (dtype == SSLA_DT_BF16 && a.dk > 32 && a.dv > 32 && wide_inputs(a, dtype) == 7)
        return Shape{a.dk <= 64 ? 64 : 128, 128, 1, true, 160, 3.5, 12.0};
    return with_shape(dtype, a.dk, a.dv, [](auto t, auto k, auto v) {
        constexpr int K = decltype(k)::value, V = decltype(v)::value;
        const int bytes = Tile<decltype(t), K, V>::bytes;
        return Shape{K, V, std::max(1, std::min(K * V >= 128 * 64 ? 2 : 4, (227 * 1024) / (bytes + 1024))), false, 145, 0.0, 0.0};
    });
}

// Tokens of a segment for sequences [i0, i1).  Undivided, the longest sequence
// bounds the time; divided, all resident CTAs share the work, but keys and
// values pass twice (`cost`), every segment is set up and its state goes
// through memory (`setup`: the tcgen05 form's tensor memory, barriers and first
// copies), two more launches follow one another (nothing of both to speak of in
// the other form), and a last round of CTAs is half empty.  Measured,
// microseconds undivided / in segments of 32 chunks / of 5: prompts of 4,096 to
// 511 tokens, 16 heads of 128 (bf16): 169 / 174 / 240; two of 8,192: 293 / 160 /
// 218; one of 65,537, 4 heads of 64: 1,729 / 118 / 200; eight of 25,000, 4 heads of
// 24, fp32: 2,302 / 400 / 388, and 352 in segments of 22.  A group's segments are
// a grid's depth: at most 65535.
int segment_tokens(const LinArgs& a, const Shape& sh, const std::vector<Seq>& seqs, size_t i0, size_t i1) {
    const long long per = static_cast<long long>(a.heads) * ((a.dv + sh.dv - 1) / sh.dv), slots = 148LL * sh.ctas;
    long long longest = 0, all = 0;
    for (size_t i = i0; i < i1; ++i) {
        const long long n = (seqs[i].len + kChunk - 1LL) / kChunk;
        longest = std::max(longest, n);
        all += n;
    }
    auto time_of = [&](long long step, long long segs) {
        const double share = std::ceil((all + segs * sh.setup) * per / slots);
        return std::max(step + sh.setup, share);
    };
    long long best = longest;
    double best_time = time_of(longest, static_cast<long long>(i1 - i0)) * 100;
    for (int parts = 2; parts <= 512; parts += parts < 32 ? 1 : parts / 16) {
        const long long step = (longest + parts - 1) / parts;
        if (step < 4) break;
        long long segs = 0;
        for (size_t i = i0; i < i1; ++i) segs += ((seqs[i].len + kChunk - 1LL) / kChunk + step - 1) / step;
        if (segs > 65535) break;                            // (the steps only get smaller)
        const double time = (time_of(step, segs) + (segs * per > slots ? step / 2 : 0)) * sh.cost + 100 * sh.launches;
        if (time < best_time) best = step, best_time = time;
    }
    return static_cast<int>(best == longest ? INT_MAX / 2 / kChunk * kChunk : best * kChunk);
}

int segments(const Seq& s, int tokens) { return s.len ? (s.len - 1) / tokens + 1 : 0; }

// Ends of the launch groups: at most kTable sequences (and 65535 segments, segment_tokens).
size_t group_end(const std::vector<Seq>& seqs, size_t i0) { return std::min(seqs.size(), i0 + kTable); }

}  // namespace

size_t chunk_workspace(const LinArgs& a, int dtype, const std::vector<Seq>& seqs) {
    const Shape sh = shape_of(a, dtype);
    size_t most = 0;
    for (size_t i0 = 0; i0 < seqs.size(); i0 = group_end(seqs, i0)) {
        const size_t i1 = group_end(seqs, i0);
        const int tokens = segment_tokens(a, sh, seqs, i0, i1);
        size_t n = 0;
        bool divided = false;
        for (size_t i = i0; i < i1; ++i) {
            n += segments(seqs[i], tokens);
            divided |= segments(seqs[i], tokens) > 1;
        }
        if (divided) most = std::max(most, n * a.heads * (8 + 4 * static_cast<size_t>(a.dk) * a.dv));
    }
    return most;
}

int chunk_launch(const LinArgs& a, int dtype, const std::vector<Seq>& seqs, void* workspace, cudaStream_t st) {
    const Shape sh = shape_of(a, dtype);
    const int wides = wide_inputs(a, dtype);
    for (size_t i0 = 0; i0 < seqs.size(); i0 = group_end(seqs, i0)) {
        const size_t i1 = group_end(seqs, i0);
        const int tokens = segment_tokens(a, sh, seqs, i0, i1);
        Table tab;
        tab.n = 0;
        tab.seg0[0] = 0;
        bool divided = false;
        for (size_t i = i0; i < i1; ++i) {
            if (!seqs[i].len) continue;
            const int n = segments(seqs[i], tokens), k = tab.n++;
            tab.start[k] = seqs[i].start;
            tab.len[k] = seqs[i].len;
            tab.slot[k] = seqs[i].slot;
            tab.step[k] = tokens;
            tab.seg0[k + 1] = tab.seg0[k] + n;
            divided |= n > 1;
        }
        if (!tab.n) continue;
        const int nseg = tab.seg0[tab.n];
        double* decays = static_cast<double*>(workspace);
        float* states = reinterpret_cast<float*>(decays + static_cast<size_t>(nseg) * a.heads);
        auto join = [&]() {
            k_chunk_join<<<dim3((a.dk * a.dv + 255) / 256, a.heads, tab.n), 256, 0, st>>>(a, tab, states, decays);
        };
        if (sh.tc) {
            const dim3 grid((a.dv + 127) / 128, a.heads, nseg);
            auto go = [&](auto k) {
                constexpr int K = decltype(k)::value, bytes = tc::Plan<K>::bytes;
                tc::Maps maps;
                const int tma =
                    tc::tensor_map(&maps.q, a.q, a.dk, a.heads / a.q_share, a.n_rows, a.q_head, a.q_row) &&
                    tc::tensor_map(&maps.k, a.k, a.dk, a.heads / a.k_share, a.n_rows, a.k_head, a.k_row) &&
                    tc::tensor_map(&maps.v, a.v, a.dv, a.heads, a.n_rows, a.v_head, a.v_row);
                const int out = aligned(a.out, 16) && a.out_row % 8 == 0 && a.out_head % 8 == 0 &&
                                tc::tensor_map(&maps.out, a.out, a.dv, a.heads, a.n_rows, a.out_head, a.out_row, 32);
                if (divided) {
                    allow_smem<tc::k_chunk_tc<K, false>>(bytes);
                    tc::k_chunk_tc<K, false><<<grid, tc::kTcThreads, bytes, st>>>(a, tab, maps, tma, out, states, decays);
                    join();
                }
                allow_smem<tc::k_chunk_tc<K, true>>(bytes);
                tc::k_chunk_tc<K, true><<<grid, tc::kTcThreads, bytes, st>>>(a, tab, maps, tma, out, states, decays);
                return launched("k_chunk_tc");
            };
            const int rc = sh.dk == 64 ? go(std::integral_constant<int, 64>()) : go(std::integral_constant<int, 128>());
            if (rc != SSLA_OK) return rc;
            continue;
        }
        const int rc = with_shape(dtype, a.dk, a.dv, [&](auto t, auto k, auto v) {
            using T = decltype(t);
            constexpr int K = decltype(k)::value, V = decltype(v)::value, bytes = Tile<T, K, V>::bytes;
            allow_smem<k_chunk<T, K, V, true>>(bytes);
            const dim3 grid((a.dv + V - 1) / V, a.heads, nseg);
            if (divided) {
                allow_smem<k_chunk<T, K, V, false>>(bytes);
                k_chunk<T, K, V, false><<<grid, kThreads, bytes, st>>>(a, tab, states, decays, wides);
                join();
            }
            k_chunk<T, K, V, true><<<grid, kThreads, bytes, st>>>(a, tab, states, decays, wides);
            return launched("k_chunk");
        });
        if (rc != SSLA_OK) return rc;
    }
    return SSLA_OK;
}

// Bits of the tcgen05 form's bounded waits since the last call (1: one ran out).
int chunk_status(unsigned* bits) {
    unsigned zero = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(bits, tc::g_status, sizeof *bits);
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(tc::g_status, &zero, sizeof zero);
    return e == cudaSuccess ? SSLA_OK : fail(SSLA_ERR_CUDA, "linear attention status: %s", cudaGetErrorString(e));
}

}  // namespace ops
}  // namespace ssla
