// ssla_linattn_tc.cuh -- the chunked linear attention of bf16 inputs with wide
// heads on the 5th-generation tensor cores (tcgen05); included by
// ssla_linattn_chunk.cu, whose comment gives the formulas, the splitting of
// 32-bit operands into bf16 pieces and the segments.
//
// The products are laid out so that 128 lanes of tensor memory are the value
// columns (dv) and the recurrent state never leaves the SM's registers and
// tensor memory.  With T the chunk's 64 tokens, all operands bf16, all sums
// 32-bit in tensor memory:
//     scores  [T, T]    = Q K^T                Q, K from shared memory
//     update  [dv, dk]  = V^T (wK)             V, three pieces of the decayed K
//     carried [dv, T]   = S^T Q^T              two pieces of S from tensor memory
//     inner   [dv, T]   = V^T P^T              two pieces of the decayed scores P
// and, in registers, S <- e^{G_C} S + update, out = scale (e^{G_t} carried + inner).
//
// Roles (20 warps, one CTA per SM):
//     warps 0-3    scores -> P: pieces to shared memory
//     warps 4-11   the state, half of dk each group: update -> S, pieces of S to
//                  tensor memory
//     warps 12-15  carried, inner -> out, through shared memory
//     (wK pieces to shared memory, as soon as the update before has read the
//     last ones: the state warps, and all three kinds where there are no outputs)
//     warps 18, 19 tiles into shared memory (three stages): whole chunks by TMA,
//                  a sequence's last, partial one by 16-byte copies with zeros;
//                  decay sums
//     warps 16, 17 issue the matrix instructions: update and carried; scores and
//                  inner
// Measured: eight prompts of up to 4,096 tokens, 16 heads of 128, take 166 us on
// 128 SMs (one CTA for each prompt and head), 2.6 us a chunk of the longest,
// where the chunk's products take 1,680 cycles of about 4,900; what bounds it is
// the roles' arithmetic (2,400 issue slots a chunk in each quarter of the SM)
// and the chain update -> state -> next wK -> update.
// Hence the division of labour below, loops that keep the roles' code in the
// instruction cache, and the state's pieces in tensor memory, where they cost
// no shared memory bandwidth.
// They meet at mbarriers only (and the state's warps, when all eight are done, at
// a named barrier).  Every wait is bounded: one that runs out sets
// the abort flag and a bit of the device's status word, all roles leave, and
// the tensor memory is freed.
#pragma once

namespace tc {

constexpr int kTcThreads = 640;
constexpr int kCopyThreads = 64;
constexpr int kStages = 3;                        // chunks whose tiles are in shared memory
constexpr int kSwRow = 128;                       // bytes of a swizzled row (64 values)
constexpr int kBlk = kChunk * kSwRow;             // a 64-token tile of 64 columns

__device__ unsigned g_status;                     // bits since the last ssla_linattn_status
constexpr unsigned kTimedOut = 1;

template <int DK> struct Plan {
    static constexpr int kTile = DK / 64 * kBlk;  // Q or K of one stage
    static constexpr int kVTile = 2 * kBlk;
    static constexpr int kStage = 2 * kTile + kVTile;
    static constexpr int kWk = kStages * kStage, kOwn = kWk + 3 * kTile, kOut = kOwn + (DK < 128 ? kStages * 2 * kBlk : 0), kEnd = kOut + 2 * kBlk;
    // A chunk's P takes the place of its K, which the products before have
    // read, where that is large enough.
    __host__ __device__ static constexpr int p_at(int st) { return DK < 128 ? kOwn + st * 2 * kBlk : st * kStage + kTile; }
    static constexpr int bytes = kEnd + 1024;     // + alignment slack
    // tensor memory columns
    static constexpr int kU = 0, kSc = DK, kO1 = DK + 64, kO2 = DK + 128, kS = DK + 192;
};

// A chunk's stage and the parity of its phases there, and the chunk's own parity.
struct Turn {
    int st = 0;
    uint32_t ph = 0, par = 0;
    __device__ void next() {
        par ^= 1;
        if (++st == kStages) st = 0, ph ^= 1;
    }
};

struct Side {                                     // what the roles share besides the tiles
    alignas(16) float2 g[kStages][kChunk];        // decay sums as (hi, lo)
    alignas(16) float eg[kStages][kChunk], wk[kStages][kChunk], gam[kStages];   // eg: times scale
    alignas(16) float end16[kStages][kChunk];     // decay from a token to the end of its 16
    int odd[kStages];                             // an update was not finite
    // A barrier of its own for each stage where a waiter does not hold back the
    // next phase by itself (a stage comes again only after everyone has left
    // it); the others' next phase needs every waiter's own arrival first.
    uint64_t full[kStages], empty[kStages], checked[kStages], p_full[kStages], wk_full[kStages];
    int again;                                    // bits: the state is not finite; there is a clear
    uint64_t sc_full, sc_free, o_full, o_free, wk_free[2], u_full, u_free, s_full, qs_full;
    uint32_t tmem;
    int abort;
};

// Shared memory descriptors (128-byte swizzle, version 1) of tiles made of
// 64-column blocks, kBlk apart, of 128-byte rows.  Only the low word moves.
// K-major: the columns are the contracted index.  MN-major: the rows are.
constexpr uint32_t kDescHi = 1024u >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t k_major(uint32_t tile) { return tile >> 4 & 0x3FFFu | 1u << 16; }
__device__ __forceinline__ uint32_t mn_major(uint32_t tile) { return tile >> 4 & 0x3FFFu | static_cast<uint32_t>(kBlk >> 4) << 16; }
__host__ __device__ constexpr uint32_t k_step(int ks) { return (ks / 4 * kBlk + ks % 4 * 32) >> 4; }
__host__ __device__ constexpr uint32_t mn_step(int ks) { return ks * 16 * kSwRow >> 4; }
// D f32, A and B bf16; M x N, `at` / `bt`: operand is MN-major.
__host__ __device__ constexpr uint32_t umma_idesc(int m, int n, int at, int bt) {
    return 1u << 4 | 1u << 7 | 1u << 10 | static_cast<uint32_t>(at) << 15 | static_cast<uint32_t>(bt) << 16 |
           static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
}
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
template <uint32_t ID> __device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, bool acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "r"(b), "n"(ID), "r"(static_cast<uint32_t>(acc)), "r"(kDescHi) : "memory");
}
template <uint32_t ID> __device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, bool acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "r"(b), "n"(ID), "r"(static_cast<uint32_t>(acc)), "r"(kDescHi) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void bar_init(uint64_t* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
// One arrival for the warp, after all its lanes' work.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if (threadIdx.x % 32 == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// Waits for a phase; false: give up.  A try suspends the thread for up to a
// microsecond or so, and there are 2^21 of them, seconds, before the CTA aborts.
// The lanes of a warp wait as one: what they test is one word.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, Side* s) {
    for (int i = 1 << 21; !bar_try(bar, parity); --i) {
        if (i == 0) {
            s->abort = 1;
            atomicOr(&g_status, kTimedOut);
        }
        if (*reinterpret_cast<volatile int*>(&s->abort)) return false;
    }
    return true;
}
// A last wait for the matrix unit, whether or not the CTA gave up: 100 ms at most.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
    const unsigned long long t0 = now_ns();
    while (!bar_try(bar, parity) && now_ns() - t0 < 100000000ull) {
    }
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_frag(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_frag(uint32_t addr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}
// Waits for the loads of r (its operands, so that nothing uses them earlier).
__device__ __forceinline__ void ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}
__device__ __forceinline__ void ld_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}
__device__ __forceinline__ void ld_wait(uint32_t (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
                 :: "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// 16-byte piece `ch` of row r in a tile of 64-column blocks.
__device__ __forceinline__ uint32_t piece_at(int r, int ch) {
    return static_cast<uint32_t>(ch / 8 * kBlk + r * kSwRow + ((ch % 8 ^ r % 8) << 4));
}
// The next bf16 piece of a pair, packed; what is left stays in it.
template <bool FIRST = false> __device__ __forceinline__ uint32_t take2(float2& x) {
    const uint32_t p = FIRST ? pack2_finite(x.x, x.y) : pack2(x.x, x.y);
    x = __ffma2_rn(unpack2(p), make_float2(-1.0f, -1.0f), x);
    return p;
}
// A 64-column, 64-row box of a [rows][heads][columns] tensor map.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int head, int row, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(head), "r"(row), "r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Starts the copies of rows [0, n) x [0, width) of a tile of COLS columns;
// the rest becomes zero.  Thread t's pieces are every (64 / (COLS / 8))-th
// row of one 16-byte column.
template <int COLS>
__device__ __forceinline__ void copy_tile(uint32_t dst, const __nv_bfloat16* p, long long stride, int n, int width, int t) {
    constexpr int kPer = COLS / 8, kStep = kCopyThreads / kPer;
    const int r0 = t / kPer, ch = t % kPer;
    const int have = max(0, min(16, (width - ch * 8) * 2));
    const __nv_bfloat16* src = p + r0 * stride + ch * 8;
    const long long step = kStep * stride;
#pragma unroll 2
    for (int i = 0; i < kChunk / kStep; ++i) {
        const int r = r0 + i * kStep, bytes = r < n ? have : 0;
        copy16(dst + piece_at(r, ch), bytes ? src : p, bytes);
        src += step;
    }
}

struct Maps {
    CUtensorMap q, k, v, out;
};

// A stage's K decayed to its chunk's end, as three bf16 pieces: the 16 bytes
// e, e + STEP, ... (N of them) of each.  Piece m of the chunk before (parity
// `prev`, where there is one) is overwritten once the matrix unit has read it.
template <int DK, int N, int STEP>
__device__ __forceinline__ bool put_keys(uint8_t* gen, Side& s, int st, int e, bool again, uint32_t prev) {
    using L = Plan<DK>;
    const uint8_t* K = gen + st * L::kStage + L::kTile;
    float2 f[N][4];
    uint32_t at[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = (e + i * STEP) / (DK / 8);
        at[i] = piece_at(r, (e + i * STEP) % (DK / 8));
        const uint4 u = *reinterpret_cast<const uint4*>(K + at[i]);
        const float2 w = make_float2(s.wk[st][r], s.wk[st][r]);
        f[i][0] = __fmul2_rn(unpack2(u.x), w);
        f[i][1] = __fmul2_rn(unpack2(u.y), w);
        f[i][2] = __fmul2_rn(unpack2(u.z), w);
        f[i][3] = __fmul2_rn(unpack2(u.w), w);
    }
#pragma unroll
    for (int m = 0; m < 3; ++m) {
        if (again && !bar_wait(m < 2 ? &s.wk_free[m] : &s.u_full, prev, &s)) return false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint4 o;
            o.x = take2(f[i][0]); o.y = take2(f[i][1]); o.z = take2(f[i][2]); o.w = take2(f[i][3]);
            *reinterpret_cast<uint4*>(gen + L::kWk + m * L::kTile + at[i]) = o;
        }
    }
    to_async();
    warp_arrive(&s.wk_full[st]);
    return true;
}

__device__ __forceinline__ void stmatrix4_trans(uint32_t addr, const uint32_t (&r)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                 :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// Piece `ch` (16 bytes) of row t of an output warp's [64][32] tile, 64-byte swizzle.
__device__ __forceinline__ uint32_t out_piece(int t, int ch) { return static_cast<uint32_t>(t * 64 + ((ch ^ (t >> 1 & 3)) << 4)); }

// Apart, like what follows: in place it cost every call 1 %.
__device__ __noinline__ void chunk_scan(const LinArgs& a, int h, long long row0, int count, int* again) {
    if (some_clear(a, h, row0, count, threadIdx.x - 128, 256)) atomicOr(again, 2);
}
// The CTA's tokens again, one by one, by warps 4 to 11.  (Everything is found anew, and the code is apart: both would
// take registers from what runs every time.)
template <int DK, bool OUT>
__device__ __noinline__ void chunk_again(const LinArgs& a, const Table& tab, float* seg_state, double* seg_decay, float* mem) {
    const int z = blockIdx.z, h = blockIdx.y, tid = threadIdx.x - 128;
    int seq = 0;
    while (tab.seg0[seq + 1] <= z) ++seq;
    const int seg = z - tab.seg0[seq], nseg = tab.seg0[seq + 1] - tab.seg0[seq], first = seg * tab.step[seq];
    const int count = min(tab.len[seq] - first, tab.step[seq]), slot = tab.slot[seq];
    const long long row0 = static_cast<long long>(tab.start[seq]) + first;
    const size_t head_state = static_cast<size_t>(a.dk) * a.dv;
    const float* from = nullptr;
    float* to = nullptr;
    if (OUT && nseg > 1) from = seg_state + (static_cast<size_t>(first_state_of(tab, seq, seg)) * a.heads + h) * head_state;
    else if (OUT && slot >= 0) from = a.state + (static_cast<size_t>(slot) * a.heads + h) * head_state;
    if (!OUT) to = seg_state + (static_cast<size_t>(z) * a.heads + h) * head_state;
    else if (seg == nseg - 1 && slot >= 0) to = a.state + (static_cast<size_t>(slot) * a.heads + h) * head_state;
    static_assert(walk_floats<DK, 128, 2, true> * 4 <= Plan<DK>::kEnd, "shared memory");
    const double total = walk<__nv_bfloat16, DK, 128, 2, OUT, true>(a, h, row0, count, blockIdx.x * 128, tid, from, to, mem,
                                                                    [] { asm volatile("bar.sync 1, 256;" ::: "memory"); });
    if (!OUT && tid == 0 && blockIdx.x == 0) seg_decay[static_cast<size_t>(z) * a.heads + h] = total;
}

template <int DK, bool OUT>
__global__ void __launch_bounds__(kTcThreads, 1)
k_chunk_tc(const __grid_constant__ LinArgs a, const __grid_constant__ Table tab, const __grid_constant__ Maps maps, int use_tma, int tma_out, float* seg_state,
           double* seg_decay) {
    using L = Plan<DK>;
    using T = __nv_bfloat16;
    constexpr int HC = DK / 2;                    // state columns of a state group
    extern __shared__ uint8_t tc_raw[];
    __shared__ Side s;
    const uint32_t base = (smem_addr(tc_raw) + 1023) & ~1023u;
    uint8_t* const gen = tc_raw + (base - smem_addr(tc_raw));
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int h = blockIdx.y, c0 = blockIdx.x * 128, width = min(128, a.dv - c0);

    int lo = 0, hi = tab.n;
    while (hi - lo > 1) {
        const int m = (lo + hi) / 2;
        if (tab.seg0[m] <= static_cast<int>(blockIdx.z)) lo = m;
        else hi = m;
    }
    const int seq = lo, seg = blockIdx.z - tab.seg0[seq], nseg = tab.seg0[seq + 1] - tab.seg0[seq];
    if (!OUT && seg == nseg - 1) return;          // (before any tensor memory is taken)
    const int first = seg * tab.step[seq], count = min(tab.len[seq] - first, tab.step[seq]);
    const int chunks = (count + kChunk - 1) / kChunk;
    const long long row0 = static_cast<long long>(tab.start[seq]) + first;
    const int slot = tab.slot[seq];
    const size_t head_state = static_cast<size_t>(a.dk) * a.dv;
    // pieces of wK: the state warps' first kOwnKeys, then the others'
    constexpr int kKeys = kChunk * DK / 8, kOwnKeys = OUT ? kKeys : kKeys / 2, kOwn = kOwnKeys / 256, kRest = kKeys / 2 / 256;

    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            bar_init(&s.full[i], 3);              // two copying warps, the decay sums
            bar_init(&s.empty[i], OUT ? 18 : 17); // the matrix unit, the state, P and output warps
            bar_init(&s.checked[i], 8);
            bar_init(&s.p_full[i], 4);
            bar_init(&s.wk_full[i], OUT ? 8 : 16);
        }
        bar_init(&s.sc_full, 1); bar_init(&s.sc_free, 4);
        bar_init(&s.o_full, 1); bar_init(&s.o_free, 4);
        bar_init(&s.wk_free[0], 1); bar_init(&s.wk_free[1], 1); bar_init(&s.u_full, 1); bar_init(&s.u_free, 8); bar_init(&s.s_full, 8); bar_init(&s.qs_full, 1);
        s.again = 0;
        s.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 18) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // value columns from 64 on that no copy writes
    if (width <= 64)
        for (int i = tid; i < kStages * kBlk / 16; i += kTcThreads)
            *reinterpret_cast<uint4*>(gen + i / (kBlk / 16) * L::kStage + 2 * L::kTile + kBlk + i % (kBlk / 16) * 16) =
                make_uint4(0, 0, 0, 0);
    to_async();
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tm = s.tmem;

    // Registers go from the small roles to the state's: launched with 96 a
    // thread (640 x 96 = 61,440), then 80, 120, 120, 96 and 56 a warpgroup
    // (60,416).
    if (warp < 4) {
        // ---- scores -> P; wK ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        const int ra = warp * 16 + lane / 4, rb = ra + 8, t2 = lane % 4 * 2;
        Turn at;
        for (int c = 0; c < chunks; ++c, at.next()) {
            const int st = at.st;
            const uint32_t par = at.par;
            if (!bar_wait(&s.full[st], at.ph, &s)) break;
            if constexpr (!OUT) {
                if (!put_keys<DK, kRest, 256>(gen, s, st, kOwnKeys + tid, c > 0, par ^ 1)) break;
            } else {
                const float2 ga = s.g[st][ra], gb = s.g[st][rb];
                if (!bar_wait(&s.sc_full, par, &s)) break;
                // (where P takes K's place, its pieces have been made by all warps)
                if (DK == 128 && !bar_wait(&s.wk_full[st], at.ph, &s)) break;
                after_sync();
                uint8_t* const pa = gen + L::p_at(st) + ra * kSwRow + t2 * 2;
                // 16 x 16 tiles: below the diagonal, on it, above it (loops not
                // unrolled: the roles' code has to stay in the instruction cache)
                const uint32_t sc = tm + (static_cast<uint32_t>(warp * 32) << 16) + L::kSc;
                uint32_t ahead[8];
                tmem_ld_frag(sc, ahead);
                ld_wait(ahead);
#pragma unroll 1
                for (int tile = 0; tile < 4; ++tile) {
                    uint8_t* const to0 = pa + ((tile * 2 ^ ra % 8) << 4);        // (rb is the same row of its atom)
                    uint8_t* const to1 = pa + ((tile * 2 + 1 ^ ra % 8) << 4);
                    if (tile > warp) {
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                *reinterpret_cast<uint32_t*>(to0 + m * kBlk + e * 8 * kSwRow) = 0;
                                *reinterpret_cast<uint32_t*>(to1 + m * kBlk + e * 8 * kSwRow) = 0;
                            }
                        continue;
                    }
                    uint32_t r[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) r[i] = ahead[i];
                    float2 x[2], y[2];                            // rows ra, rb of the tile's two column groups
                    if (tile < warp) {
                        tmem_ld_frag(sc + (tile + 1) * 16, ahead);
                        // below the diagonal: the decay to the end of the columns' 16 tokens, times that from there
                        const float2 ge = s.g[st][tile * 16 + 15];
                        const float ea = exp2_fast((ga.x - ge.x) + (ga.y - ge.y)) * a.scale;
                        const float eb = exp2_fast((gb.x - ge.x) + (gb.y - ge.y)) * a.scale;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float2 e = *reinterpret_cast<const float2*>(&s.end16[st][tile * 16 + j * 8 + t2]);
                            x[j] = __fmul2_rn(make_float2(__uint_as_float(r[j * 4]), __uint_as_float(r[j * 4 + 1])),
                                              __fmul2_rn(e, make_float2(ea, ea)));
                            y[j] = __fmul2_rn(make_float2(__uint_as_float(r[j * 4 + 2]), __uint_as_float(r[j * 4 + 3])),
                                              __fmul2_rn(e, make_float2(eb, eb)));
                        }
                    } else {
                        before_sync();
                        warp_arrive(&s.sc_free);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int col = tile * 16 + j * 8 + t2;
                            const float4 g = *reinterpret_cast<const float4*>(&s.g[st][col]);
                            const float e0 = exp2_fast((ga.x - g.x) + (ga.y - g.y)), e1 = exp2_fast((ga.x - g.z) + (ga.y - g.w));
                            const float f0 = exp2_fast((gb.x - g.x) + (gb.y - g.y)), f1 = exp2_fast((gb.x - g.z) + (gb.y - g.w));
                            x[j].x = col <= ra ? __uint_as_float(r[j * 4]) * (e0 * a.scale) : 0.0f;
                            x[j].y = col + 1 <= ra ? __uint_as_float(r[j * 4 + 1]) * (e1 * a.scale) : 0.0f;
                            y[j].x = col <= rb ? __uint_as_float(r[j * 4 + 2]) * (f0 * a.scale) : 0.0f;
                            y[j].y = col + 1 <= rb ? __uint_as_float(r[j * 4 + 3]) * (f1 * a.scale) : 0.0f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint8_t* const to = j ? to1 : to0;
                        *reinterpret_cast<uint32_t*>(to) = take2<true>(x[j]);
                        *reinterpret_cast<uint32_t*>(to + kBlk) = pack2(x[j].x, x[j].y);
                        *reinterpret_cast<uint32_t*>(to + 8 * kSwRow) = take2<true>(y[j]);
                        *reinterpret_cast<uint32_t*>(to + 8 * kSwRow + kBlk) = pack2(y[j].x, y[j].y);
                    }
                    ld_wait(ahead);
                }
                to_async();
                warp_arrive(&s.p_full[st]);
            }
            warp_arrive(&s.empty[st]);
        }
    } else if (warp < 12) {
        // ---- the state: value column d, dk columns [k0, k0 + HC) ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
        const int wg = (warp - 4) / 4, quad = warp % 4, d = quad * 32 + lane, k0 = wg * HC;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        float2 S[HC / 2];
        const float* from = nullptr;
        if (OUT && nseg > 1) from = seg_state + (static_cast<size_t>(first_state_of(tab, seq, seg)) * a.heads + h) * head_state;
        else if (OUT && slot >= 0) from = a.state + (static_cast<size_t>(slot) * a.heads + h) * head_state;
        {
            const bool there = from && d < width;
            const float* p = there ? from + static_cast<size_t>(k0) * a.dv + c0 + d : nullptr;
            int left = there ? a.dk - k0 : 0;
#pragma unroll
            for (int i = 0; i < HC / 2; ++i) {
                S[i].x = left > 0 ? *p : 0.0f;
                p += a.dv;
                S[i].y = left > 1 ? *p : 0.0f;
                p += a.dv;
                left -= 2;
            }
        }
        auto put_pieces = [&]() {                  // S as two bf16 pieces, two columns a word
#pragma unroll
            for (int b = 0; b < HC / 16; ++b) {
                uint32_t big[8], small[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float2 x = S[b * 8 + i];
                    big[i] = take2<true>(x);
                    small[i] = pack2(x.x, x.y);
                }
                tmem_st8(tm + lanes + L::kS + k0 / 2 + b * 8, big);
                tmem_st8(tm + lanes + L::kS + DK / 2 + k0 / 2 + b * 8, small);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            before_sync();
            warp_arrive(&s.s_full);
        };
        Turn keys, at;                             // of chunk c, of chunk c - 1
        for (int c = 0; c <= chunks; ++c) {
            const bool more = c < chunks;
            if (more) {
                if (!bar_wait(&s.full[keys.st], keys.ph, &s)) break;
                if (!put_keys<DK, kOwn, 256>(gen, s, keys.st, tid - 128, c > 0, keys.par ^ 1)) break;
                keys.next();
            }
            if (c) {
                const int st = at.st;
                const float2 gam = make_float2(s.gam[st], s.gam[st]);
                if (!bar_wait(&s.u_full, at.par, &s)) break;
                after_sync();
                bool odd = false;
#pragma unroll
                for (int b = 0; b < HC / 16; ++b) {
                    uint32_t u[16];
                    tmem_ld16(tm + lanes + L::kU + k0 + b * 16, u);
                    ld_wait(u);
                    // every column of this lane has every v of value column d as a factor
                    if (b == 0) odd = (u[0] & 0x7F800000u) == 0x7F800000u;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        S[b * 8 + i] = __ffma2_rn(gam, S[b * 8 + i],
                                                  make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])));
                }
                before_sync();
                warp_arrive(&s.u_free);
                if (OUT) {
                    if (odd) s.odd[st] = 1;
                    warp_arrive(&s.checked[st]);
                }
                warp_arrive(&s.empty[st]);
                if (OUT && more && !bar_wait(&s.qs_full, at.par, &s)) break;
                at.next();
            }
            if (OUT && more) {
                after_sync();
                put_pieces();
            }
        }
        float* to = nullptr;
        if (!OUT) to = seg_state + (static_cast<size_t>(blockIdx.z) * a.heads + h) * head_state;
        else if (seg == nseg - 1 && slot >= 0) to = a.state + (static_cast<size_t>(slot) * a.heads + h) * head_state;
        // Not finite, and a clear among the decays: all of it again at the end.  (The eight warps all come here,
        // whatever they waited for in vain.)
        float2 zero[4] = {};
#pragma unroll
        for (int i = 0; i < HC / 2; ++i) zero[i % 4] = __ffma2_rn(S[i], make_float2(0.0f, 0.0f), zero[i % 4]);   // NaN where one is not finite
        const float2 all = __fadd2_rn(__fadd2_rn(zero[0], zero[1]), __fadd2_rn(zero[2], zero[3]));
        if (all.x + all.y != 0.0f) atomicOr(&s.again, 1);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (s.again) {
            chunk_scan(a, h, row0, count, &s.again);
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        if (to && d < width && s.again != 3) {
            float* p = to + static_cast<size_t>(k0) * a.dv + c0 + d;
            int left = a.dk - k0;
#pragma unroll
            for (int i = 0; i < HC / 2; ++i) {
                if (left > 0) *p = S[i].x;
                p += a.dv;
                if (left > 1) *p = S[i].y;
                p += a.dv;
                left -= 2;
            }
        }
    } else if (warp < 16) {
        // ---- carried, inner -> out: 32 value columns a warp, 64 tokens; wK ----
        const int ow = warp - 12, d = ow * 32 + lane, cols = min(32, width - ow * 32);
        const uint32_t lanes = static_cast<uint32_t>(ow * 32) << 16;
        Turn keys, at;                             // of chunk c, of chunk c - 1
        for (int c = 0; c <= chunks; ++c) {
            if (!OUT && c < chunks) {
                if (!bar_wait(&s.full[keys.st], keys.ph, &s)) break;
                if (!put_keys<DK, kRest, 256>(gen, s, keys.st, kOwnKeys + tid - 256, c > 0, keys.par ^ 1)) break;
                warp_arrive(&s.empty[keys.st]);
                keys.next();
            }
            if (OUT && c) {
                const int st = at.st, done = c - 1, n = min(kChunk, count - done * kChunk);
                const uint32_t par = at.par;
                if (!bar_wait(&s.full[st], at.ph, &s) || !bar_wait(&s.checked[st], at.ph, &s)) break;
                const bool odd = s.odd[st] != 0;
                if (!bar_wait(&s.qs_full, par, &s)) break;
                if (!bar_wait(&s.o_full, par, &s)) break;
                after_sync();
                at.next();
                // the last chunk's store has read the tile
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
                uint8_t* const tile = gen + L::kOut + ow * (kChunk * 64);
                const uint32_t tile_at = smem_addr(tile);
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {            // 16 value columns
                    uint32_t r[32], u[32];
                    tmem_ld_frag(tm + lanes + (static_cast<uint32_t>(half * 16) << 16) + L::kO1, r);
                    tmem_ld_frag(tm + lanes + (static_cast<uint32_t>(half * 16) << 16) + L::kO2, u);
                    ld_wait(r);
                    ld_wait(u);
                    if (half == 1 && !odd) {
                        before_sync();
                        warp_arrive(&s.o_free);
                    }
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {              // tokens j * 8 .. + 16
                        uint32_t m[4];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float2 e = *reinterpret_cast<const float2*>(&s.eg[st][(j + i) * 8 + lane % 4 * 2]);
                            const uint32_t *x = r + (j + i) * 4, *z = u + (j + i) * 4;
                            const float2 y0 = __ffma2_rn(e, make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])),
                                                         make_float2(__uint_as_float(z[0]), __uint_as_float(z[1])));
                            const float2 y1 = __ffma2_rn(e, make_float2(__uint_as_float(x[2]), __uint_as_float(x[3])),
                                                         make_float2(__uint_as_float(z[2]), __uint_as_float(z[3])));
                            m[2 * i] = pack2(y0.x, y0.y);
                            m[2 * i + 1] = pack2(y1.x, y1.y);
                        }
                        // matrices: (tokens j, columns 0-7), (j, 8-15), (j + 1, 0-7), (j + 1, 8-15)
                        stmatrix4_trans(tile_at + out_piece((j + lane / 16) * 8 + lane % 8, half * 2 + lane / 8 % 2), m);
                    }
                }
                __syncwarp();
                if (odd) {
                    // A value in this chunk was not finite: if it is in this lane's column, the product with
                    // masked zeros has reached the tokens before it.  Their inner sums again, one by one.
                    const uint8_t* V = gen + st * L::kStage + 2 * L::kTile;
                    const uint8_t* P = gen + L::p_at(st);
                    auto value = [&](int t) {
                        return __bfloat162float(*reinterpret_cast<const T*>(V + piece_at(t, d / 8) + d % 8 * 2));
                    };
                    int bad = 0;
                    while (bad < n && finite(value(bad))) ++bad;
                    for (int i = 0; i < n; ++i) {
                        uint32_t o1;
                        __syncwarp();
                        asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(o1) : "r"(tm + lanes + L::kO1 + i));
                        asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(o1) :: "memory");
                        if (bad == n) continue;
                        float inner = __int_as_float(0x7FC00000);
                        if (i < bad) {
                            inner = 0.0f;
                            for (int t = 0; t <= i; ++t) {
                                const uint32_t at_p = piece_at(i, t / 8) + t % 8 * 2;
                                inner = fmaf(__bfloat162float(*reinterpret_cast<const T*>(P + at_p)) +
                                                 __bfloat162float(*reinterpret_cast<const T*>(P + kBlk + at_p)),
                                             value(t), inner);
                            }
                        }
                        *reinterpret_cast<T*>(tile + out_piece(i, lane / 8) + lane % 8 * 2) =
                            __float2bfloat16_rn(fmaf(s.eg[st][i], __uint_as_float(o1), inner));
                    }
                    before_sync();
                    warp_arrive(&s.o_free);
                }
                const long long row = row0 + static_cast<long long>(done) * kChunk;
                to_async();                        // before the store reads the tile
                warp_arrive(&s.empty[st]);
                if (cols > 0 && tma_out && n == kChunk) {
                    if (lane == 0) {
                        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];"
                                     :: "l"(&maps.out), "r"(c0 + ow * 32), "r"(h), "r"(static_cast<int>(row)), "r"(tile_at) : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else if (cols > 0) {
                    T* const p = static_cast<T*>(a.out) + row * a.out_row + h * a.out_head + c0 + ow * 32;
                    for (int i = lane; i < n * 4; i += 32) {
                        const int t = i / 4, ch = i % 4;
                        const uint8_t* from = tile + out_piece(t, ch);
                        T* to = p + t * a.out_row + ch * 8;
                        if (tma_out && ch * 8 + 8 <= cols) {
                            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
                        } else {
                            for (int j = 0; j < 8; ++j)
                                if (ch * 8 + j < cols) to[j] = reinterpret_cast<const T*>(from)[j];
                        }
                    }
                }
            }
        }
        if (OUT && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    } else if (warp >= 18) {
        // ---- tiles; decay sums (warp 18), the next chunk's values in flight ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        const int t = lane + (warp - 18) * 32, hq = h / a.q_share, hk = h / a.k_share;
        const T* Q = static_cast<const T*>(a.q) + hq * a.q_head + row0 * a.q_row;
        const T* K = static_cast<const T*>(a.k) + hk * a.k_head + row0 * a.k_row;
        const T* V = static_cast<const T*>(a.v) + h * a.v_head + c0 + row0 * a.v_row;
        double total = 0.0;
        bool cleared = false;                      // (this lane's tokens)
        float2 g = make_float2(0.0f, 0.0f);
        if (warp == 18) g = chunk_decay_values(a, row0, min(kChunk, count), h, lane);
        Turn at;
        for (int c = 0; c < chunks; ++c, at.next()) {
            const int n = min(kChunk, count - c * kChunk), st = at.st;
            if (c >= kStages && !bar_wait(&s.empty[st], at.ph ^ 1, &s)) break;
            uint64_t* const bar = &s.full[st];
            const uint32_t to = base + st * L::kStage;
            const bool tma = use_tma && n == kChunk;
            if (!tma) {
                const long long row = static_cast<long long>(c) * kChunk;
                copy_tile<DK>(to + L::kTile, K + row * a.k_row, a.k_row, n, a.dk, t);
                copy_tile<128>(to + 2 * L::kTile, V + row * a.v_row, a.v_row, n, width, t);
                if (OUT) copy_tile<DK>(to, Q + row * a.q_row, a.q_row, n, a.dk, t);
                asm volatile("cp.async.commit_group;" ::: "memory");
            } else if (warp == 18 && elect()) {
                const int row = static_cast<int>(row0) + c * kChunk;
                const uint32_t bytes = ((OUT ? 2 : 1) * (DK / 64) + (width > 64 ? 2 : 1)) * kBlk;
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
#pragma unroll
                for (int b = 0; b < DK / 64; ++b) tma_box(to + L::kTile + b * kBlk, &maps.k, b * 64, hk, row, bar);
                tma_box(to + 2 * L::kTile, &maps.v, c0, h, row, bar);
                if (width > 64) tma_box(to + 2 * L::kTile + kBlk, &maps.v, c0 + 64, h, row, bar);
                if (OUT)
#pragma unroll
                    for (int b = 0; b < DK / 64; ++b) tma_box(to + b * kBlk, &maps.q, b * 64, hq, row, bar);
            }
            __syncwarp();
            if (warp == 18) {
                float2 ahead = make_float2(0.0f, 0.0f);
                if (c + 1 < chunks)
                    ahead = chunk_decay_values(a, row0 + (c + 1LL) * kChunk, min(kChunk, count - (c + 1) * kChunk), h, lane);
                const DecaySums d = chunk_decays(g, lane);
                if (!OUT) cleared |= g.x == -INFINITY || g.y == -INFINITY;
                total += d.total;
                *reinterpret_cast<float4*>(&s.g[st][2 * lane]) = make_float4(d.hi[0], d.lo[0], d.hi[1], d.lo[1]);
                *reinterpret_cast<float2*>(&s.eg[st][2 * lane]) = make_float2(d.grown[0] * a.scale, d.grown[1] * a.scale);
                *reinterpret_cast<float2*>(&s.wk[st][2 * lane]) = make_float2(d.left[0], d.left[1]);
                const float hi16 = __shfl_sync(0xFFFFFFFFu, d.hi[1], lane | 7), lo16 = __shfl_sync(0xFFFFFFFFu, d.lo[1], lane | 7);
                *reinterpret_cast<float2*>(&s.end16[st][2 * lane]) =
                    make_float2(exp2_fast((hi16 - d.hi[0]) + (lo16 - d.lo[0])), exp2_fast((hi16 - d.hi[1]) + (lo16 - d.lo[1])));
                if (lane == 0) s.gam[st] = d.whole, s.odd[st] = 0;
                warp_arrive(bar);
                g = ahead;
            }
            if (!tma) {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                to_async();
            }
            if (!tma || warp == 19) warp_arrive(bar);
        }
        if (!OUT && warp == 18) {
            if (__any_sync(0xFFFFFFFFu, cleared)) total = -INFINITY;
            if (lane == 0 && blockIdx.x == 0) seg_decay[static_cast<size_t>(blockIdx.z) * a.heads + h] = total;
        }
    } else if (warp == 16) {
        // ---- matrix instructions of the state: update, carried (the warp as one, one lane issues) ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        constexpr uint32_t id_u = umma_idesc(128, DK, 1, 1), id_q = umma_idesc(128, 64, 0, 0);
        const uint32_t wk_desc = mn_major(base + L::kWk);
        Turn at;
        for (int c = 0; c < chunks; ++c, at.next()) {
            const uint32_t par = at.par, tiles = base + at.st * L::kStage;
            const uint32_t q = k_major(tiles), v = mn_major(tiles + 2 * L::kTile);
            if (!bar_wait(&s.full[at.st], at.ph, &s)) break;
            if (c && !bar_wait(&s.u_free, par ^ 1, &s)) break;
            if (!bar_wait(&s.wk_full[at.st], at.ph, &s)) break;
            after_sync();
            if (elect()) {
#pragma unroll
                for (int m = 0; m < 3; ++m) {
#pragma unroll
                    for (int i = 0; i < kChunk / 16; ++i)
                        umma_ss<id_u>(tm + L::kU, v + mn_step(i), wk_desc + (m * L::kTile >> 4) + mn_step(i), i + m > 0);
                    commit(m < 2 ? &s.wk_free[m] : &s.u_full);
                }
                if (!OUT) commit(&s.empty[at.st]);
            }
            __syncwarp();
            if constexpr (OUT) {
                if (c && !bar_wait(&s.o_free, par ^ 1, &s)) break;
                if (!bar_wait(&s.s_full, par, &s)) break;
                after_sync();
                if (elect()) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int i = 0; i < DK / 16; ++i)
                            umma_ts<id_q>(tm + L::kO1, tm + L::kS + m * (DK / 2) + i * 8, q + k_step(i), m + i > 0);
                    commit(&s.qs_full);
                    commit(&s.empty[at.st]);
                }
                __syncwarp();
            }
        }
        // nothing of this warp's may be in flight when the CTA frees its tensor memory
        drain(&s.u_full, (chunks - 1) & 1);
        if (OUT) drain(&s.qs_full, (chunks - 1) & 1);
    } else {
        // ---- matrix instructions of the chunk itself: scores, inner ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if constexpr (OUT) {
            constexpr uint32_t id_sc = umma_idesc(64, 64, 0, 0), id_p = umma_idesc(128, 64, 1, 0);
            auto scores = [&](int st) {
                const uint32_t q = k_major(base + st * L::kStage), k = k_major(base + st * L::kStage + L::kTile);
                if (elect()) {
#pragma unroll
                    for (int i = 0; i < DK / 16; ++i) umma_ss<id_sc>(tm + L::kSc, q + k_step(i), k + k_step(i), i > 0);
                    commit(&s.sc_full);
                }
                __syncwarp();
            };
            bool ok = bar_wait(&s.full[0], 0, &s);
            after_sync();
            if (ok) scores(0);
            Turn at;
            for (int c = 0; ok && c < chunks; ++c) {
                const int st = at.st;
                const uint32_t par = at.par, v = mn_major(base + st * L::kStage + 2 * L::kTile);
                const uint32_t p_desc = k_major(base + L::p_at(st)), ph = at.ph;
                at.next();
                if (c + 1 < chunks) {              // the next scores first, so that P follows P
                    if (!(ok = bar_wait(&s.full[at.st], at.ph, &s))) break;
                    if (!(ok = bar_wait(&s.sc_free, par, &s))) break;
                    after_sync();
                    scores(at.st);
                }
                if (c && !(ok = bar_wait(&s.o_free, par ^ 1, &s))) break;
                if (!(ok = bar_wait(&s.p_full[st], ph, &s))) break;
                after_sync();
                if (elect()) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int i = 0; i < kChunk / 16; ++i)
                            umma_ss<id_p>(tm + L::kO2, v + mn_step(i), p_desc + (m * kBlk >> 4) + k_step(i), m + i > 0);
                    commit(&s.o_full);
                    commit(&s.empty[st]);
                }
                __syncwarp();
            }
            drain(&s.o_full, (chunks - 1) & 1);
        }
    }
    __syncwarp();
    before_sync();
    __syncthreads();
    if (s.again == 3) {                           // by the state's warps, whose registers are enough for it
        if (warp >= 12 && warp < 16 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;\n\tfence.proxy.async;" ::: "memory");
        __syncthreads();
        if (warp >= 4 && warp < 12) chunk_again<DK, OUT>(a, tab, seg_state, seg_decay, reinterpret_cast<float*>(gen));
    }
    if (warp == 18) {
        after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm));
    }
}

// ---- host ----
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {
    static const EncodeTiled f = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return reinterpret_cast<EncodeTiled>(fn);
    }();
    return f;
}

// The map of a [rows][heads][width] bf16 tensor in boxes of `cols` columns (64:
// 128-byte swizzle, 32: 64-byte) and 64 rows of one head, zeros beyond the width.  false: not a tensor TMA takes
// (a broadcast stride); its tiles go by 16-byte copies.
inline bool tensor_map(CUtensorMap* m, const void* p, int width, int heads, int rows, long long head, long long row,
                       int cols = 64) {
    if ((heads > 1 && head <= 0) || (rows > 1 && row <= 0) || !encode_tiled()) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(std::max(heads > 1 ? head : 8LL, 8LL)) * 2,
                                   static_cast<cuuint64_t>(std::max(rows > 1 ? row : 8LL, 8LL)) * 2};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(cols), 1, kChunk}, one[3] = {1, 1, 1};
    return encode_tiled()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, one,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tc
