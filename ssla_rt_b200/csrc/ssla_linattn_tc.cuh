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
// Roles (16 warps, one CTA per SM):
//     warps 0-3    scores -> P (pieces to shared memory); carried, inner -> out
//     warps 4-11   the state, half of dk each group: wK pieces to shared memory,
//                  update -> S, pieces of S to tensor memory
//     warps 12-13  tiles into shared memory (three stages), non-finite v
//     warp 14      decay sums
//     warp 15      issues the matrix instructions
// They meet at mbarriers only.  Every wait is bounded: one that runs out sets
// the abort flag and a bit of the device's status word, all roles leave, and
// the tensor memory is freed.
#pragma once

namespace tc {

constexpr int kTcThreads = 512;                    // 128 registers a thread
constexpr int kCopyWarps = 2, kCopyThreads = 32 * kCopyWarps;
constexpr int kStages = 3;                        // chunks whose tiles are in shared memory
constexpr int kSwRow = 128;                       // bytes of a swizzled row (64 values)
constexpr int kBlk = kChunk * kSwRow;             // a 64-token tile of 64 columns

__device__ unsigned g_status;                     // bits since the last ssla_linattn_status
constexpr unsigned kTimedOut = 1;

template <int DK> struct Plan {
    static constexpr int kTile = DK / 64 * kBlk;  // Q or K of one stage
    static constexpr int kVTile = 2 * kBlk;
    static constexpr int kStage = 2 * kTile + kVTile;
    static constexpr int kWk = kStages * kStage, kP = kWk + 3 * kTile, kEnd = kP + 2 * kBlk;
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
    float ghi[kStages][kChunk], glo[kStages][kChunk], eg[kStages][kChunk], wk[kStages][kChunk], gam[kStages];
    int bad[kStages][kCopyWarps][128], any[kStages][kCopyWarps];                // first non-finite row by column, as each copying warp saw it
    uint64_t full[kStages], empty[kStages], sc_full, sc_free, p_full, o_full, o_free, wk_full, u_full, u_free, s_full, qs_full;
    uint32_t tmem;
    int abort;

    __device__ bool any_bad(int st) const { return (any[st][0] | any[st][1]) != 0; }
    __device__ int first_bad(int st, int d) const {
        return min(bad[st][0][d], bad[st][1][d]);
    }
};

__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    // 128-byte swizzle, version 1
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | static_cast<uint64_t>((lead >> 4) & 0x3FFFu) << 16 |
           static_cast<uint64_t>((stride >> 4) & 0x3FFFu) << 32 | 1ull << 46 | 2ull << 61;
}
// 64-column blocks of rows one after the other: columns are the contracted
// index (K-major), or the rows are (MN-major, blocks kBlk apart).
__device__ __forceinline__ uint64_t k_major(uint32_t tile, int ks) {
    return umma_desc(tile + ks / 4 * kBlk + ks % 4 * 32, 16, 1024);
}
__device__ __forceinline__ uint64_t mn_major(uint32_t tile, int ks) { return umma_desc(tile + ks * 16 * kSwRow, kBlk, 1024); }
// D f32, A and B bf16; M x N, `at` / `bt`: operand is MN-major.
__host__ __device__ constexpr uint32_t umma_idesc(int m, int n, int at, int bt) {
    return 1u << 4 | 1u << 7 | 1u << 10 | static_cast<uint32_t>(at) << 15 | static_cast<uint32_t>(bt) << 16 |
           static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(id), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(id), "r"(acc) : "memory");
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
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// Waits for a phase, two seconds at most; false: give up.
__device__ __forceinline__ bool lane_wait(uint64_t* bar, uint32_t parity, Side* s) {
    if (bar_try(bar, parity)) return true;
    const unsigned long long t0 = now_ns();
    while (!bar_try(bar, parity)) {
        if (*reinterpret_cast<volatile int*>(&s->abort)) return false;
        if (now_ns() - t0 > 2000000000ull) {
            *reinterpret_cast<volatile int*>(&s->abort) = 1;
            atomicOr(&g_status, kTimedOut);
            return false;
        }
    }
    return true;
}
// The same for a whole warp, which goes on or gives up as one.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, Side* s) {
    return __all_sync(0xFFFFFFFFu, lane_wait(bar, parity, s));
}
// A last wait for the matrix unit, whether or not the CTA gave up: 100 ms at most.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
    const unsigned long long t0 = now_ns();
    while (!bar_try(bar, parity) && now_ns() - t0 < 100000000ull) {
    }
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
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
// Waits for the loads of r (its operands, so that nothing uses them earlier).
__device__ __forceinline__ void ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// 16-byte piece `ch` of row r in a tile of 64-column blocks.
__device__ __forceinline__ uint32_t piece_at(int r, int ch) {
    return static_cast<uint32_t>(ch / 8 * kBlk + r * kSwRow + ((ch % 8 ^ r % 8) << 4));
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
#pragma unroll
    for (int i = 0; i < kChunk / kStep; ++i) {
        const int r = r0 + i * kStep, bytes = r < n ? have : 0;
        copy16(dst + piece_at(r, ch), bytes ? src : p, bytes);
        src += step;
    }
}

template <int DK, bool OUT>
__global__ void __launch_bounds__(kTcThreads, 1)
k_chunk_tc(LinArgs a, const __grid_constant__ Table tab, float* seg_state, double* seg_decay) {
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

    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            bar_init(&s.full[i], kCopyWarps + 1);
            bar_init(&s.empty[i], OUT ? 13 : 9);  // the matrix unit, the state warps, the output warps
        }
        bar_init(&s.sc_full, 1); bar_init(&s.sc_free, 4); bar_init(&s.p_full, 4);
        bar_init(&s.o_full, 1); bar_init(&s.o_free, 4); bar_init(&s.wk_full, 8);
        bar_init(&s.u_full, 1); bar_init(&s.u_free, 8); bar_init(&s.s_full, 8); bar_init(&s.qs_full, 1);
        s.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 15) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    before_sync();
    __syncthreads();
    after_sync();
    const uint32_t tm = s.tmem;

    if (warp < 4) {
        // ---- scores -> P; carried, inner -> out ----
        if constexpr (OUT) {
            const int ra = warp * 16 + lane / 4, rb = ra + 8, t2 = lane % 4 * 2;
            const int d = warp * 32 + lane;       // value column of the outputs
            const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
            Turn at;
            for (int c = 0; c < chunks; ++c, at.next()) {
                const int st = at.st, n = min(kChunk, count - c * kChunk);
                if (!bar_wait(&s.full[st], at.ph, &s)) break;
                if (!bar_wait(&s.sc_full, at.par, &s)) break;
                after_sync();
                uint32_t r[32];
                tmem_ld_frag(tm + lanes + L::kSc, r);
                const float ha = s.ghi[st][ra], la = s.glo[st][ra], hb = s.ghi[st][rb], lb = s.glo[st][rb];
                ld_wait(r);
                before_sync();
                warp_arrive(&s.sc_free);
                uint8_t* const pa = gen + L::kP + ra * kSwRow + t2 * 2;
                uint8_t* const pb = pa + 8 * kSwRow;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float x[4] = {};
                    if (j * 8 <= warp * 16 + 15) {                // not wholly above the diagonal
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int col = j * 8 + t2 + e;
                            const float hs = s.ghi[st][col], ls = s.glo[st][col];
                            if (col <= ra) x[e] = __uint_as_float(r[j * 4 + e]) * exp2f((ha - hs) + (la - ls));
                            if (col <= rb) x[2 + e] = __uint_as_float(r[j * 4 + 2 + e]) * exp2f((hb - hs) + (lb - ls));
                        }
                    }
                    const int ch = (j ^ ra % 8) << 4;             // (rb is the same row of its atom)
                    *reinterpret_cast<uint32_t*>(pa + ch) = take(x[0], x[1]);
                    *reinterpret_cast<uint32_t*>(pa + kBlk + ch) = take(x[0], x[1]);
                    *reinterpret_cast<uint32_t*>(pb + ch) = take(x[2], x[3]);
                    *reinterpret_cast<uint32_t*>(pb + kBlk + ch) = take(x[2], x[3]);
                }
                to_async();
                warp_arrive(&s.p_full);
                if (!bar_wait(&s.o_full, at.par, &s)) break;
                after_sync();
                const bool any = s.any_bad(st);
                const int from = any ? s.first_bad(st, d) : kChunk;
                T* p = static_cast<T*>(a.out) + (row0 + c * kChunk) * a.out_row + h * a.out_head + c0 + d;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t u[32];
                    tmem_ld32(tm + lanes + L::kO1 + half * 32, r);
                    tmem_ld32(tm + lanes + L::kO2 + half * 32, u);
                    ld_wait(r);
                    ld_wait(u);
                    if (half == 1) {
                        before_sync();
                        warp_arrive(&s.o_free);
                    }
                    const int left = n - half * 32;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float y = fmaf(s.eg[st][half * 32 + i], __uint_as_float(r[i]), __uint_as_float(u[i])) * a.scale;
                        if (any && half * 32 + i >= from) y = __int_as_float(0x7FC00000);
                        if (i < left && d < width) *p = __float2bfloat16_rn(y);
                        p += a.out_row;
                    }
                }
                warp_arrive(&s.empty[st]);
            }
        }
    } else if (warp < 12) {
        // ---- the state: value column d, dk columns [k0, k0 + HC) ----
        const int wg = (warp - 4) / 4, quad = warp % 4, d = quad * 32 + lane, k0 = wg * HC, me = tid - 128;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        float S[HC];
        const float* from = nullptr;
        if (OUT && seg > 0) from = seg_state + (static_cast<size_t>(blockIdx.z - 1) * a.heads + h) * head_state;
        else if (OUT && slot >= 0) from = a.state + (static_cast<size_t>(slot) * a.heads + h) * head_state;
#pragma unroll
        for (int i = 0; i < HC; ++i)
            S[i] = from && d < width && k0 + i < a.dk ? from[static_cast<size_t>(k0 + i) * a.dv + c0 + d] : 0.0f;
        auto put_pieces = [&]() {                  // S as two bf16 pieces, two columns a word
#pragma unroll
            for (int b = 0; b < HC / 32; ++b) {
                uint32_t hi16[16], lo16[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float x = S[b * 32 + 2 * i], y = S[b * 32 + 2 * i + 1];
                    hi16[i] = take(x, y);
                    lo16[i] = pack2(x, y);
                }
                tmem_st16(tm + lanes + L::kS + k0 / 2 + b * 16, hi16);
                tmem_st16(tm + lanes + L::kS + DK / 2 + k0 / 2 + b * 16, lo16);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            before_sync();
            warp_arrive(&s.s_full);
        };
        auto put_keys = [&](int st) {              // a stage's K decayed to the chunk's end, three pieces
            const uint8_t* K = gen + st * L::kStage + L::kTile;
#pragma unroll
            for (int i = 0; i < kChunk * DK / 8 / 256; ++i) {
                const int e = me + i * 256, r = e / (DK / 8), ch = e % (DK / 8);
                const uint32_t at = piece_at(r, ch);
                const uint4 u = *reinterpret_cast<const uint4*>(K + at);
                const float w = s.wk[st][r];
                float2 f[4] = {unpack2(u.x), unpack2(u.y), unpack2(u.z), unpack2(u.w)};
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j].x *= w, f[j].y *= w;
#pragma unroll
                for (int m = 0; m < 3; ++m) {
                    uint4 o;
                    o.x = take(f[0].x, f[0].y); o.y = take(f[1].x, f[1].y);
                    o.z = take(f[2].x, f[2].y); o.w = take(f[3].x, f[3].y);
                    *reinterpret_cast<uint4*>(gen + L::kWk + m * L::kTile + at) = o;
                }
            }
            to_async();
            warp_arrive(&s.wk_full);
        };
        if (OUT) put_pieces();
        bool ok = bar_wait(&s.full[0], 0, &s);
        if (ok) put_keys(0);
        Turn at;
        for (int c = 0; ok && c < chunks; ++c) {
            const int st = at.st;
            const uint32_t par = at.par;
            if (!(ok = bar_wait(&s.u_full, par, &s))) break;
            after_sync();
            const float gam = s.gam[st];
#pragma unroll
            for (int b = 0; b < HC / 32; ++b) {
                uint32_t u[32];
                tmem_ld32(tm + lanes + L::kU + k0 + b * 32, u);
                ld_wait(u);
#pragma unroll
                for (int i = 0; i < 32; ++i) S[b * 32 + i] = fmaf(gam, S[b * 32 + i], __uint_as_float(u[i]));
            }
            before_sync();
            warp_arrive(&s.u_free);
            if (s.any_bad(st) && s.first_bad(st, d) < kChunk)
#pragma unroll
                for (int i = 0; i < HC; ++i) S[i] = __int_as_float(0x7FC00000);
            warp_arrive(&s.empty[st]);
            at.next();
            if (c + 1 < chunks) {
                if (!(ok = bar_wait(&s.full[at.st], at.ph, &s))) break;
                put_keys(at.st);
                if (OUT) {
                    if (!(ok = bar_wait(&s.qs_full, par, &s))) break;
                    after_sync();
                    put_pieces();
                }
            }
        }
        float* to = nullptr;
        if (!OUT) to = seg_state + (static_cast<size_t>(blockIdx.z) * a.heads + h) * head_state;
        else if (seg == nseg - 1 && slot >= 0) to = a.state + (static_cast<size_t>(slot) * a.heads + h) * head_state;
        if (to && d < width)
#pragma unroll
            for (int i = 0; i < HC; ++i)
                if (k0 + i < a.dk) to[static_cast<size_t>(k0 + i) * a.dv + c0 + d] = S[i];
    } else if (warp < 12 + kCopyWarps) {
        // ---- tiles, non-finite values ----
        const int t = tid - 384, w = warp - 12;
        const T* Q = static_cast<const T*>(a.q) + (h / a.q_share) * a.q_head + row0 * a.q_row;
        const T* K = static_cast<const T*>(a.k) + (h / a.k_share) * a.k_head + row0 * a.k_row;
        const T* V = static_cast<const T*>(a.v) + h * a.v_head + c0 + row0 * a.v_row;
        Turn at, arrived;
        bool ok = true;
        // chunk c's copies start as soon as its stage is free; then chunk c - 1,
        // whose copies started a chunk's time earlier, is handed over
        for (int c = 0; ok && c <= chunks; ++c) {
            if (c < chunks) {
                const int n = min(kChunk, count - c * kChunk);
                if (c >= kStages && !(ok = bar_wait(&s.empty[at.st], at.ph ^ 1, &s))) break;
                const uint32_t to = base + at.st * L::kStage;
                const long long row = static_cast<long long>(c) * kChunk;
                copy_tile<DK>(to + L::kTile, K + row * a.k_row, a.k_row, n, a.dk, t);
                copy_tile<128>(to + 2 * L::kTile, V + row * a.v_row, a.v_row, n, width, t);
                if (OUT) copy_tile<DK>(to, Q + row * a.q_row, a.q_row, n, a.dk, t);
#pragma unroll
                for (int i = 0; i < 4; ++i) s.bad[at.st][w][lane + 32 * i] = kChunk;
                if (lane == 0) s.any[at.st][w] = 0;
                __syncwarp();
                at.next();
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (c == 0) continue;
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            uint8_t* const tile = gen + arrived.st * L::kStage + 2 * L::kTile;
            bool any = false;
#pragma unroll
            for (int i = 0; i < kChunk * 16 / kCopyThreads; ++i) {       // the pieces this thread has copied
                const int r = t / 16 + i * (kCopyThreads / 16), ch = t % 16;
                const uint4 u = *reinterpret_cast<const uint4*>(tile + piece_at(r, ch));
                bool odd = false;
                for (uint32_t x : {u.x, u.y, u.z, u.w}) odd |= (x & 0x7F80u) == 0x7F80u || (x & 0x7F800000u) == 0x7F800000u;
                if (odd) {
                    uint16_t* p = reinterpret_cast<uint16_t*>(tile + piece_at(r, ch));
                    any = true;
                    for (int j = 0; j < 8; ++j)
                        if ((p[j] & 0x7F80u) == 0x7F80u) {
                            p[j] = 0;
                            atomicMin(&s.bad[arrived.st][w][ch * 8 + j], r);
                        }
                }
            }
            if (any) s.any[arrived.st][w] = 1;
            to_async();
            warp_arrive(&s.full[arrived.st]);
            arrived.next();
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == 14) {
        // ---- decay sums, the next chunk's values in flight ----
        double total = 0.0;
        Turn at;
        float2 g = chunk_decay_values(a, row0, min(kChunk, count), h, lane);
        for (int c = 0; c < chunks; ++c, at.next()) {
            float2 ahead = make_float2(0.0f, 0.0f);
            if (c + 1 < chunks)
                ahead = chunk_decay_values(a, row0 + (c + 1LL) * kChunk, min(kChunk, count - (c + 1) * kChunk), h, lane);
            if (c >= kStages && !bar_wait(&s.empty[at.st], at.ph ^ 1, &s)) break;
            const int st = at.st;
            total += chunk_decays(g, lane, s.ghi[st], s.glo[st], s.eg[st], s.wk[st], &s.gam[st]);
            warp_arrive(&s.full[st]);
            g = ahead;
        }
        if (!OUT && lane == 0 && blockIdx.x == 0) seg_decay[static_cast<size_t>(blockIdx.z) * a.heads + h] = total;
    } else if (lane == 0) {
        // ---- matrix instructions ----
        constexpr uint32_t id_sc = umma_idesc(64, 64, 0, 0), id_u = umma_idesc(128, DK, 1, 1), id_q = umma_idesc(128, 64, 0, 0),
                           id_p = umma_idesc(128, 64, 1, 0);
        const int ksteps = (a.dk + 15) / 16;       // of the contraction over dk
        auto scores = [&](int st) {
            const uint32_t q = base + st * L::kStage;
            for (int k = 0; k < ksteps; ++k) umma_ss(tm + L::kSc, k_major(q, k), k_major(q + L::kTile, k), id_sc, k > 0);
            commit(&s.sc_full);
        };
        bool ok = lane_wait(&s.full[0], 0, &s);
        after_sync();
        if (OUT && ok) scores(0);
        Turn at;
        for (int c = 0; ok && c < chunks; ++c) {
            const uint32_t par = at.par, prev = par ^ 1, tiles = base + at.st * L::kStage, v = tiles + 2 * L::kTile;
            const int st = at.st;
            if (!(ok = lane_wait(&s.wk_full, par, &s))) break;
            if (c && !(ok = lane_wait(&s.u_free, prev, &s))) break;
            after_sync();
            for (int k = 0; k < kChunk / 16; ++k)
                for (int m = 0; m < 3; ++m)
                    umma_ss(tm + L::kU, mn_major(v, k), mn_major(base + L::kWk + m * L::kTile, k), id_u, k + m > 0);
            commit(&s.u_full);
            if constexpr (OUT) {
                if (!(ok = lane_wait(&s.s_full, par, &s))) break;
                if (c && !(ok = lane_wait(&s.o_free, prev, &s))) break;
                after_sync();
                for (int m = 0; m < 2; ++m)
                    for (int k = 0; k < ksteps; ++k)
                        umma_ts(tm + L::kO1, tm + L::kS + m * (DK / 2) + k * 8, k_major(tiles, k), id_q, m + k > 0);
                commit(&s.qs_full);
                if (!(ok = lane_wait(&s.p_full, par, &s))) break;
                after_sync();
                for (int m = 0; m < 2; ++m)
                    for (int k = 0; k < kChunk / 16; ++k)
                        umma_ss(tm + L::kO2, mn_major(v, k), k_major(base + L::kP + m * kBlk, k), id_p, m + k > 0);
                commit(&s.o_full);
            }
            commit(&s.empty[st]);
            at.next();
            if (OUT && c + 1 < chunks) {
                if (!(ok = lane_wait(&s.full[at.st], at.ph, &s))) break;
                if (!(ok = lane_wait(&s.sc_free, par, &s))) break;
                after_sync();
                scores(at.st);
            }
        }
        // nothing of this CTA's may be in flight when it frees its tensor memory
        drain(&s.u_full, (chunks - 1) & 1);
        if (OUT) drain(&s.o_full, (chunks - 1) & 1);
    }
    __syncwarp();
    before_sync();
    __syncthreads();
    if (warp == 15) {
        after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm));
    }
}

}  // namespace tc
