// ssla_linattn.cu -- linear attention with a decay per head
// (include/ssla_ops.h): S <- e^g S + k v^T, out = scale S^T q, with a 32-bit
// state S [dk][dv] per head.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <new>
#include <vector>

#include "ssla_linattn.cuh"

namespace ssla {
namespace ops {
namespace {

// ---------------------------------------------------------------------------
// One token per row: a CTA holds a head's state columns [c0, c0 + 32) in
// registers and applies the rows that name its slot.  Memory bound: the state
// is read and written once, 8 dk dv bytes; everything a token needs is asked
// for together with the state, before the slots are compared, and the state
// leaves before the output is summed up.  256 rows of 16 heads of 128 x 128:
// 94 us, 89% of the measured copy rate (105 us without the streaming hints).
//
// Thread (tx, rg): columns c0 + tx * VEC .. + VEC, state rows rg + i * RG.
// ---------------------------------------------------------------------------
constexpr int kStepThreads = 128;
constexpr int kStepCols = 32;

template <typename T, int VEC, int RPT>
struct StepTile {
    static constexpr int TX = kStepCols / VEC, RG = kStepThreads / TX;
    float s[RPT][VEC], kk[RPT], qq[RPT], vv[VEC], g;
    int tx, rg, c0;
    bool live;                                     // this thread's columns exist

    __device__ void place(const LinArgs& a) {
        tx = threadIdx.x % TX;
        rg = threadIdx.x / TX;
        c0 = blockIdx.x * kStepCols + tx * VEC;
        live = c0 < a.dv;
    }
    __device__ float* at(const LinArgs& a, int slot, int h) const {
        return a.state + (static_cast<size_t>(slot) * a.heads + h) * a.dk * a.dv + c0;
    }
    __device__ void load(const LinArgs& a, int slot, int h) {
        const float* p = at(a, slot, h);
#pragma unroll
        for (int i = 0; i < RPT; ++i)
            if (live && rg + i * RG < a.dk)
                load_vec_hint<float, VEC>(p + static_cast<size_t>(rg + i * RG) * a.dv, s[i], a.stream);
    }
    __device__ void store(const LinArgs& a, int slot, int h) const {
        float* p = at(a, slot, h);
#pragma unroll
        for (int i = 0; i < RPT; ++i)
            if (live && rg + i * RG < a.dk)
                store_vec_hint<float, VEC>(p + static_cast<size_t>(rg + i * RG) * a.dv, s[i], a.stream);
    }
    __device__ void fetch(const LinArgs& a, int row, int h) {
        const T* q = static_cast<const T*>(a.q) + row * a.q_row + (h / a.q_share) * a.q_head;
        const T* k = static_cast<const T*>(a.k) + row * a.k_row + (h / a.k_share) * a.k_head;
        const T* v = static_cast<const T*>(a.v) + row * a.v_row + h * a.v_head;
        g = a.decay[row * a.decay_row + h * a.decay_head];
#pragma unroll
        for (int j = 0; j < VEC; ++j) vv[j] = live ? to_f<T>(v[c0 + j]) : 0.0f;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int r = rg + i * RG;
            kk[i] = r < a.dk ? to_f<T>(k[r]) : 0.0f;
            qq[i] = r < a.dk ? to_f<T>(q[r]) : 0.0f;
        }
    }
    // The fetched token: updates the state, and leaves its output's parts in o.
    __device__ void apply(const LinArgs& a, float (&o)[VEC]) {
        const float e = expf(g);
        if (g == -INFINITY)                        // clears the state, NaN and infinities in it too
#pragma unroll
            for (int i = 0; i < RPT; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) s[i][j] = 0.0f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < RPT; ++i)
            if (rg + i * RG < a.dk)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    s[i][j] = fmaf(kk[i], vv[j], e * s[i][j]);
                    o[j] = fmaf(qq[i], s[i][j], o[j]);
                }
    }
    // Sums the parts over the row groups (lanes of a warp with the same tx,
    // then the warps) and writes the output columns.
    __device__ void output(const LinArgs& a, int row, int h, float (&o)[VEC], float* red) {
#pragma unroll
        for (int m = TX; m < 32; m <<= 1)
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] += __shfl_xor_sync(0xFFFFFFFFu, o[j], m);
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane < TX)
#pragma unroll
            for (int j = 0; j < VEC; ++j) red[warp * kStepCols + tx * VEC + j] = o[j];
        __syncthreads();
        const int c = blockIdx.x * kStepCols + threadIdx.x;
        if (threadIdx.x < kStepCols && c < a.dv) {
            float t = 0.0f;
#pragma unroll
            for (int w = 0; w < kStepThreads / 32; ++w) t += red[w * kStepCols + threadIdx.x];
            static_cast<T*>(a.out)[row * a.out_row + h * a.out_head + c] = from_f<T>(t * a.scale);
        }
        __syncthreads();
    }
};

template <typename T, int VEC, int RPT>
__global__ void __launch_bounds__(kStepThreads) k_linattn_step(LinArgs a, const int* __restrict__ slots) {
    using Tile = StepTile<T, VEC, RPT>;
    __shared__ float red[kStepThreads / 32 * kStepCols];
    __shared__ int next_s;
    Tile t;
    t.place(a);
    const int h = blockIdx.y;
    int row = blockIdx.z;
    const int slot = slots ? slots[row] : row;
    if (slot < 0 || slot >= a.n_slots) {           // padding row
        const int c = blockIdx.x * kStepCols + threadIdx.x;
        if (threadIdx.x < kStepCols && c < a.dv)
            static_cast<T*>(a.out)[row * a.out_row + h * a.out_head + c] = from_f<T>(0.0f);
        return;
    }
    t.load(a, slot, h);
    t.fetch(a, row, h);
    for (;;) {
        int next = INT_MAX, before = 0;
        if (slots) {
            // rows that name this slot: the first of them applies all, in row order
            if (threadIdx.x == 0) next_s = INT_MAX;
            for (int r = threadIdx.x; r < a.n_rows; r += kStepThreads)
                if (r != row && slots[r] == slot) {
                    if (r < row) before = 1;
                    else next = min(next, r);
                }
            before = row == static_cast<int>(blockIdx.z) ? __syncthreads_or(before) : (__syncthreads(), 0);
            if (before) return;
            if (next != INT_MAX) atomicMin(&next_s, next);
            __syncthreads();
            next = next_s;
        }
        float o[VEC];
        t.apply(a, o);
        if (next == INT_MAX) t.store(a, slot, h);
        t.output(a, row, h, o, red);
        if (next == INT_MAX) break;
        row = next;
        t.fetch(a, row, h);
    }
}

// ---- host ----------------------------------------------------------------

// The state rows of a thread, by dk and the vector width.  (CTAs of 64 columns
// and 256 threads were slower: 114 us against 105 for 256 rows of 16 heads of
// 128 x 128.)
template <typename F> int with_tile(int dtype, bool vec4, int dk, F&& f) {
    using std::integral_constant;
    auto by_rows = [&](auto t, auto v) {
        constexpr int V = decltype(v)::value, RG = 4 * V;
        if (dk <= 2 * RG) return f(t, v, integral_constant<int, 2>());
        if (dk <= 4 * RG) return f(t, v, integral_constant<int, 4>());
        if (dk <= 8 * RG) return f(t, v, integral_constant<int, 8>());
        if constexpr (V == 1) {
            if (dk <= 16 * RG) return f(t, v, integral_constant<int, 16>());
            return f(t, v, integral_constant<int, 32>());
        }
        return fail(SSLA_ERR_ARG, "dk %d", dk);
    };
    auto by_vec = [&](auto t) {
        return vec4 ? by_rows(t, integral_constant<int, 4>()) : by_rows(t, integral_constant<int, 1>());
    };
    return dtype == SSLA_DT_F32 ? by_vec(float()) : dtype == SSLA_DT_BF16 ? by_vec(__nv_bfloat16()) : by_vec(__half());
}

struct Span {                       // bytes that a strided [rows][heads][width] tensor spans
    const void* p;
    size_t n;
};

Span span_of(const void* p, long long row, long long head, int n_rows, int heads, int width, int size) {
    if (n_rows == 0) return {p, 0};
    return {p, static_cast<size_t>((n_rows - 1) * row + (heads - 1) * head + width) * size};
}

// Checks everything of `a` but the sequences / slots; SSLA_OK or an error.
int check_args(const SslaLinAttn* a, const char* who, bool need_state) {
    if (!a) return fail(SSLA_ERR_ARG, "%s: null argument", who);
    if (!dtype_ok(a->dtype)) return fail(SSLA_ERR_ARG, "%s: dtype %d is not an SSLA_DT_* value", who, a->dtype);
    if (a->n_rows > INT_MAX - 65536) return fail(SSLA_ERR_ARG, "%s: %d rows, at most 2^31 - 2^16", who, a->n_rows);
    if (a->n_rows < 0 || a->n_slots < 0) return fail(SSLA_ERR_ARG, "%s: negative n_rows or n_slots", who);
    if (a->heads < 1 || a->heads > 65535 || a->q_heads < 1 || a->k_heads < 1 || a->heads % a->q_heads ||
        a->heads % a->k_heads)
        return fail(SSLA_ERR_ARG, "%s: heads %d must be 1..65535 and a multiple of q_heads %d and k_heads %d", who,
                    a->heads, a->q_heads, a->k_heads);
    if (a->dk < 1 || a->dk > SSLA_LINATTN_MAX_DK || a->dv < 1 || a->dv > SSLA_LINATTN_MAX_DV)
        return fail(SSLA_ERR_ARG, "%s: dk %d must be 1..%d and dv %d must be 1..%d", who, a->dk, SSLA_LINATTN_MAX_DK,
                    a->dv, SSLA_LINATTN_MAX_DV);
    if (!std::isfinite(a->scale)) return fail(SSLA_ERR_ARG, "%s: scale is not finite", who);
    if (a->n_rows == 0) return SSLA_OK;
    if (!a->q || !a->k || !a->v || !a->out || !a->decay || (need_state && !a->state))
        return fail(SSLA_ERR_ARG, "%s: null pointer", who);
    const long long most = LLONG_MAX / 16 / std::max(a->n_rows, a->heads);
    for (long long s : {a->q_row, a->q_head, a->k_row, a->k_head, a->v_row, a->v_head, a->out_row, a->out_head,
                        a->decay_row, a->decay_head})
        if (s < 0 || s > most) return fail(SSLA_ERR_ARG, "%s: a stride is negative or too large", who);
    const int sz = dtype_size(a->dtype);
    if (!aligned(a->q, sz) || !aligned(a->k, sz) || !aligned(a->v, sz) || !aligned(a->out, sz) ||
        !aligned(a->decay, 4) || !aligned(a->state, 4))
        return fail(SSLA_ERR_ARG, "%s: a pointer is not aligned to its element", who);
    // no two outputs share a place
    const bool rows_outer = (a->heads == 1 || a->out_head >= a->dv) &&
                            (a->n_rows == 1 || a->out_row >= (a->heads - 1) * a->out_head + a->dv);
    const bool heads_outer = (a->n_rows == 1 || a->out_row >= a->dv) &&
                             (a->heads == 1 || a->out_head >= (a->n_rows - 1) * a->out_row + a->dv);
    if (!rows_outer && !heads_outer) return fail(SSLA_ERR_ARG, "%s: out overlaps itself", who);
    const Span out = span_of(a->out, a->out_row, a->out_head, a->n_rows, a->heads, a->dv, sz);
    const Span st = {a->state, static_cast<size_t>(a->state ? a->n_slots : 0) * a->heads * a->dk * a->dv * 4};
    const Span in[4] = {span_of(a->q, a->q_row, a->q_head, a->n_rows, a->q_heads, a->dk, sz),
                        span_of(a->k, a->k_row, a->k_head, a->n_rows, a->k_heads, a->dk, sz),
                        span_of(a->v, a->v_row, a->v_head, a->n_rows, a->heads, a->dv, sz),
                        span_of(a->decay, a->decay_row, a->decay_head, a->n_rows, a->heads, 1, 4)};
    for (const Span& s : in)
        if (overlaps(out.p, out.n, s.p, s.n) || overlaps(st.p, st.n, s.p, s.n))
            return fail(SSLA_ERR_ARG, "%s: out or state overlaps an input", who);
    if (overlaps(out.p, out.n, st.p, st.n)) return fail(SSLA_ERR_ARG, "%s: out overlaps state", who);
    return SSLA_OK;
}

// Whether [p, p + n) meets a tensor of the (checked) call; `written` ones only, or all.
bool meets(const SslaLinAttn* a, const void* p, size_t n, bool written) {
    const int sz = dtype_size(a->dtype);
    auto in = [&](const Span& s) { return overlaps(p, n, s.p, s.n); };
    if (in(span_of(a->out, a->out_row, a->out_head, a->n_rows, a->heads, a->dv, sz)) ||
        in({a->state, static_cast<size_t>(a->state ? a->n_slots : 0) * a->heads * a->dk * a->dv * 4}))
        return true;
    return !written && (in(span_of(a->q, a->q_row, a->q_head, a->n_rows, a->q_heads, a->dk, sz)) ||
                        in(span_of(a->k, a->k_row, a->k_head, a->n_rows, a->k_heads, a->dk, sz)) ||
                        in(span_of(a->v, a->v_row, a->v_head, a->n_rows, a->heads, a->dv, sz)) ||
                        in(span_of(a->decay, a->decay_row, a->decay_head, a->n_rows, a->heads, 1, 4)));
}

LinArgs device_args(const SslaLinAttn* a) {
    LinArgs d;
    d.q = a->q; d.k = a->k; d.v = a->v; d.out = a->out; d.decay = a->decay; d.state = a->state;
    d.q_row = a->q_row; d.q_head = a->q_head; d.k_row = a->k_row; d.k_head = a->k_head;
    d.v_row = a->v_row; d.v_head = a->v_head; d.out_row = a->out_row; d.out_head = a->out_head;
    d.decay_row = a->decay_row; d.decay_head = a->decay_head;
    d.n_rows = a->n_rows; d.heads = a->heads; d.q_share = a->heads / a->q_heads; d.k_share = a->heads / a->k_heads;
    d.dk = a->dk; d.dv = a->dv; d.n_slots = a->n_slots; d.scale = a->scale;
    d.stream = 8LL * a->n_rows * a->heads * a->dk * a->dv > kStreamBytes;   // the step's state traffic
    return d;
}

bool state_vec4(const SslaLinAttn* a) { return a->dv % 4 == 0 && aligned(a->state, 16); }

// The sequences of a chunked call, checked against each other and the rows,
// and, with `slotted`, their slots.
int check_seqs(const SslaLinAttn* a, const int* offsets, const int* lengths, bool slotted, const int* slots, int n_seq,
               std::vector<Seq>& out) {
    const char* who = "linear attention";
    if (n_seq < 0 || (n_seq > 0 && !offsets)) return fail(SSLA_ERR_ARG, "%s: no offsets", who);
    out.reserve(n_seq);
    bool any_slot = false;
    for (int i = 0; i < n_seq; ++i) {
        const long long len = lengths ? lengths[i] : static_cast<long long>(offsets[i + 1]) - offsets[i];
        if (offsets[i] < 0 || len < 0 || offsets[i] + len > a->n_rows)
            return fail(SSLA_ERR_ARG, "%s: sequence %d is rows [%d, %lld) of %d", who, i, offsets[i], offsets[i] + len,
                        a->n_rows);
        const int slot = !slotted ? -1 : slots ? slots[i] : i;
        if (slot < -1 || slot >= a->n_slots) {
            if (a->state || slots) return fail(SSLA_ERR_ARG, "%s: slot %d of %d", who, slot, a->n_slots);
        }
        out.push_back({offsets[i], static_cast<int>(len), a->state ? slot : -1});
        any_slot |= slots && slot >= 0;
    }
    if (any_slot && !a->state) return fail(SSLA_ERR_ARG, "%s: slots without a state", who);
    std::vector<Seq> s(out);
    if (lengths) {                                  // plain offsets cannot overlap
        std::sort(s.begin(), s.end(), [](const Seq& x, const Seq& y) { return x.start < y.start; });
        long long end = 0;
        for (const Seq& x : s) {
            if (!x.len) continue;
            if (x.start < end) return fail(SSLA_ERR_ARG, "%s: sequences overlap at row %d", who, x.start);
            end = static_cast<long long>(x.start) + x.len;
        }
    }
    if (slots) {
        std::sort(s.begin(), s.end(), [](const Seq& x, const Seq& y) { return x.slot < y.slot; });
        for (size_t i = 1; i < s.size(); ++i)
            if (s[i].slot >= 0 && s[i].slot == s[i - 1].slot)
                return fail(SSLA_ERR_ARG, "%s: slot %d occurs twice", who, s[i].slot);
    }
    return SSLA_OK;
}

}  // namespace
}  // namespace ops
}  // namespace ssla

using namespace ssla::ops;

extern "C" {

int ssla_linattn_step(const SslaLinAttn* a, const int* slots, void* stream) {
    const char* who = "linear attention step";
    if (const int rc = check_args(a, who, true); rc != SSLA_OK) return rc;
    if (a->n_rows > 65535) return fail(SSLA_ERR_ARG, "%s: %d rows, at most 65535", who, a->n_rows);
    if (!slots && a->n_rows > a->n_slots)
        return fail(SSLA_ERR_ARG, "%s: %d rows for %d slots", who, a->n_rows, a->n_slots);
    if (!aligned(slots, 4)) return fail(SSLA_ERR_ARG, "%s: slots are not aligned", who);
    if (a->n_rows == 0) return SSLA_OK;
    if (slots && meets(a, slots, 4ull * a->n_rows, true)) return fail(SSLA_ERR_ARG, "%s: out or state overlaps slots", who);
    OnDevice dev(a->device);
    if (dev.err != SSLA_OK) return dev.err;
    const LinArgs d = device_args(a);
    return with_tile(a->dtype, state_vec4(a), a->dk, [&](auto t, auto v, auto r) {
        const dim3 grid((a->dv + kStepCols - 1) / kStepCols, a->heads, a->n_rows);
        k_linattn_step<decltype(t), decltype(v)::value, decltype(r)::value>
            <<<grid, kStepThreads, 0, static_cast<cudaStream_t>(stream)>>>(d, slots);
        return launched("k_linattn_step");
    });
}

int ssla_linattn_chunk_workspace(const SslaLinAttn* a, const int* offsets, const int* lengths, int n_seq,
                                 size_t* bytes) {
    if (!bytes) return fail(SSLA_ERR_ARG, "linear attention: null argument");
    if (const int rc = check_args(a, "linear attention", false); rc != SSLA_OK) return rc;
    try {
        std::vector<Seq> seqs;
        if (const int rc = check_seqs(a, offsets, lengths, false, nullptr, n_seq, seqs); rc != SSLA_OK) return rc;
        *bytes = a->n_rows ? chunk_workspace(device_args(a), a->dtype, seqs) : 0;
        return SSLA_OK;
    } catch (const std::exception&) {
        return fail(SSLA_ERR_CUDA, "linear attention: host allocation failed");
    }
}

int ssla_linattn_chunk(const SslaLinAttn* a, const int* offsets, const int* lengths, const int* slots, int n_seq,
                       void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "linear attention";
    if (const int rc = check_args(a, who, false); rc != SSLA_OK) return rc;
    try {
        std::vector<Seq> seqs;
        if (const int rc = check_seqs(a, offsets, lengths, true, slots, n_seq, seqs); rc != SSLA_OK) return rc;
        if (a->n_rows == 0 || seqs.empty()) return SSLA_OK;
        const LinArgs d = device_args(a);
        const size_t need = chunk_workspace(d, a->dtype, seqs);
        if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
            return fail(SSLA_ERR_ARG, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", who, workspace_bytes, need);
        if (need && meets(a, workspace, need, false)) return fail(SSLA_ERR_ARG, "%s: the workspace overlaps a tensor", who);
        OnDevice dev(a->device);
        if (dev.err != SSLA_OK) return dev.err;
        return chunk_launch(d, a->dtype, seqs, workspace, static_cast<cudaStream_t>(stream));
    } catch (const std::exception&) {
        return fail(SSLA_ERR_CUDA, "%s: host allocation failed", who);
    }
}

int ssla_linattn_status(int device, unsigned* status) {
    if (!status) return fail(SSLA_ERR_ARG, "linear attention status: null argument");
    OnDevice dev(device);
    if (dev.err != SSLA_OK) return dev.err;
    return chunk_status(status);
}

}  // extern "C"
