// The loss of a refit: a student's logits against the alternatives a teacher gave, with the
// gradient of the weighted losses from the same reading of the logits.
//
// With p = softmax(x / T) and K kept columns (given, inside the row, no repeat of an earlier one):
//   renorm: q = softmax(l / T) over the kept;           loss = sum q_k (log q_k - log p_k)
//           dx_i = w/T (Q p_i - [i kept] q_i),          Q = 1 (0 if nothing is kept)
//   rest:   q_k = e^l_k, q_r = 1 - sum q_k for all other columns together, p_r their sum of p;
//           loss = sum q_k (log q_k - log p_k) + q_r (log q_r - log p_r)
//           kept: dx = w (Q p_k - q_k);  others: dx_i = w (Q p_r - q_r) p_i / p_r,  Q = sum q_k + q_r.
// p_r is a sum of its own and not 1 - sum p_k, which has no digits left where the student
// agrees with the teacher: the kept columns are taken out of the running sums by a bitmap of
// the part in LDS, and p_i / p_r is the softmax over the others, so nothing overflows where
// p_r does not fit float32 either.
//
// Bound by reading the logits once and writing the gradient once.  A part of a row (256 lanes of 8
// vectors) stays in a workgroup's registers while the row's parts tell each other their sums, and
// is written from there: every logit is read once, and with 6 workgroups on a CU the others load or
// store while one waits.  The row's first part finishes it: it alone looks up the student's logits at
// the teacher's columns (64 lines a row) and writes the gradient there, so the other parts leave
// those columns out.  4096 x 131072 bf16 with 64 alternatives: 424 us, 5.1 TB/s (a copy: 4.9).
// (A whole row in the registers of 1024 lanes leaves one workgroup a CU and nothing to do while
// it sums, 549 us; reading twice costs half again the traffic, 570 us.)
#include "logits.h"
#include "words.h"

namespace ddm {
namespace logits {

struct DistillArgs {
    const char* x;
    int64_t n, v, ld_bytes, out_ld_bytes;
    const void* index;
    int index_wide;
    const float* logprob;
    const float* weight;       // NULL: 1
    int k, rest, parts;
    float temperature;
    float* loss;
    char* out;                 // NULL: the loss alone
    uint32_t *tickets, queues; // one part a row: NULL
    uint64_t* words;           // [n][parts + 2]: m, s of a part's columns that are not kept (renorm: of
                               // all); then the row's Bulk.  The loss alone: [n][parts], no Bulk
};

// The teacher's alternatives of a row, one a lane of a wave.
struct Kept {
    int col;                   // -1: none
    float l, x;                // teacher's log probability, student's logit
};

// The column of the thread's alternative; -1: none.
__device__ __forceinline__ int column_of(const DistillArgs& a, int64_t r) {
    if ((int)threadIdx.x >= a.k) return -1;
    const int64_t i = target_at(a.index, a.index_wide, r * a.k + threadIdx.x);
    return i >= 0 && i < a.v ? (int)i : -1;
}
template <typename T>
__device__ __forceinline__ Kept load_kept(const DistillArgs& a, int64_t r, int col, const Row<T>& row) {
    const int lane = threadIdx.x & 63;
    Kept k{col, -INFINITY, -INFINITY};
    if (lane < a.k) k.l = a.logprob[r * a.k + lane];
    uint64_t same = __ballot(k.col >= 0);                // lanes of the same column, a bit of it at a time
    for (int bit = 0; bit < 19; ++bit) {
        const bool one = k.col >> bit & 1;
        const uint64_t ones = __ballot(one);
        same &= one ? ones : ~ones;
    }
    if (k.col >= 0 && (same & ((1ull << lane) - 1ull))) k.col = -1;      // the first of equal ones counts
    if (k.col >= 0)
        k.x = row.at(k.col);
    else
        k.l = -INFINITY;
    return k;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) v += __shfl_xor(v, k);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) v = fmaxf(v, __shfl_xor(v, k));
    return v;
}

// One wave: the row's loss (to a.loss), the gradient of the lane's kept column, and what every
// other column's gradient is made of: 2^((x - m) c - log2 s) * factor.
struct Bulk {
    float m, log2_s, factor;
};
template <typename T>
__device__ __forceinline__ Bulk finish_row(const DistillArgs& a, int64_t r, const Kept& k, Part p, float& kept_grad) {
    const float c = kLog2e / a.temperature;
    const bool mine = k.col >= 0;
    const float w = a.weight ? a.weight[r] : 1.0f;
    // the student
    const float m = a.rest ? fmaxf(p.m, wave_max(k.x)) : p.m;
    const float e = mine ? __builtin_amdgcn_exp2f((k.x - m) * c) : 0.0f;
    const float total = a.rest ? p.s * __builtin_amdgcn_exp2f(fmaxf((p.m - m) * c, kDead)) + wave_sum(e) : p.s;
    const bool alive = total > 0.0f, bad = total != total;
    const float log_total = __builtin_amdgcn_logf(total) * kLn2;
    const float logp = alive ? (k.x - m) / a.temperature - log_total : -INFINITY;
    const float log_rest = p.s > 0.0f ? (p.m - m) / a.temperature + __builtin_amdgcn_logf(p.s) * kLn2 - log_total : -INFINITY;
    // the teacher
    float logq = k.l, q, q_rest = 0.0f;
    if (a.rest) {
        q = mine ? expf(logq) : 0.0f;
        q_rest = 1.0f - wave_sum(q);
        // float32 log probabilities cannot tell a remainder under 2^-20 from none
        if (q_rest < 0x1p-20f || __popcll(__ballot(mine)) == a.v) q_rest = 0.0f;
    } else {
        const float z = logq / a.temperature, top = wave_max(z);
        const bool some = top > -INFINITY;
        q = mine && some ? expf(z - top) : 0.0f;
        const float qs = wave_sum(q);
        q = some ? q / qs : q;
        logq = some ? z - top - logf(qs) : z;
    }
    if (__any(mine && k.l != k.l)) q = __builtin_nanf("");
    const float whole = wave_sum(q) + q_rest;
    float loss = wave_sum(!(q <= 0.0f) ? q * (logq - logp) : 0.0f);
    if (q_rest > 0.0f) loss += q_rest * (logf(q_rest) - log_rest);
    if (bad) loss = __builtin_nanf("");
    if ((threadIdx.x & 63) == 0) a.loss[r] = loss;
    // the gradient; a row with nothing left has none
    const float scale = w / a.temperature;
    const bool none = w == 0.0f || (!alive && !bad);
    const float p_rest = alive ? __builtin_amdgcn_exp2f(log_rest * kLog2e) : 0.0f;
    kept_grad = none ? 0.0f : (__builtin_amdgcn_exp2f(logp * kLog2e) * whole - q) * scale;
    if (bad && !none) kept_grad = __builtin_nanf("");
    Bulk b;
    b.m = p.m;
    b.log2_s = p.s > 0.0f ? __builtin_amdgcn_logf(p.s) : 0.0f;
    b.factor = none ? 0.0f : bad ? __builtin_nanf("") : a.rest ? (p_rest * whole - q_rest) * scale : whole * scale;
    return b;
}

// What of a part is kept, a byte a vector.
template <int NT, int NV>
__device__ __forceinline__ void mark_kept(uint32_t* bits, bool set, int vector, int entry) {
    for (int i = threadIdx.x; i < NT * NV / 4; i += NT) bits[i] = 0;
    __syncthreads();
    if (set && vector >= 0 && vector < NT * NV) atomicOr(&bits[vector >> 2], 1u << ((vector & 3) * 8 + entry));
    __syncthreads();
}

// The running maximum and sum of a part, kept columns apart.
template <typename T, int NT, int NV>
__device__ __forceinline__ Part sum_part(const uint4 (&raw)[NV], float c, bool rest, const uint32_t* bits) {
    Lane l = no_lane();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[T::kVec];
        unpack(raw[i], f, T());
        if (rest) {
            const uint32_t b = ((const uint8_t*)bits)[i * NT + threadIdx.x];
            if (__any(b != 0)) {
#pragma unroll
                for (int e = 0; e < T::kVec; ++e) f[e] = b >> e & 1 ? -INFINITY : f[e];
            }
        }
        add_vector<false>(l, f, largest(f), c);
    }
    return part_of(l, c);
}

// The gradient of a column that is not kept: 2^(x c - shift) * factor, one fused product an entry.
// What shift = m c + log2 s loses in rounding is in the factor; where it is too large for that (see
// add_vector) the difference x - m comes first.
struct Writer {
    float m, log2_s, shift, factor;
    bool wide;
};
__device__ __forceinline__ Writer writer_of(const Bulk& b, float c) {
    Writer w{b.m, b.log2_s, fmaf(b.m, c, b.log2_s), b.factor, false};
    w.wide = !(fabsf(w.shift) < kWide);
    if (!w.wide) w.factor *= __builtin_amdgcn_exp2f(-(fmaf(b.m, c, -w.shift) + b.log2_s));
    return w;
}
template <int N>
__device__ __forceinline__ void gradient(float (&f)[N], float c, const Writer& w) {
    if (w.wide || w.factor == 0.0f) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            f[e] = w.factor == 0.0f ? 0.0f : __builtin_amdgcn_exp2f((f[e] - w.m) * c - w.log2_s) * w.factor;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = __builtin_amdgcn_exp2f(fmaf(f[e], c, -w.shift)) * w.factor;
    }
}

__device__ __forceinline__ uint64_t wait_for(const uint64_t* p) {
    uint64_t w = peek(p);
    for (uint32_t looks = 0; w == kUnset; ++looks) {
        if (looks >= *(volatile uint32_t*)&guard.looks) {
            tell_gave_up();
            break;
        }
        __builtin_amdgcn_s_sleep(1);
        w = peek(p);
    }
    return w;                                            // unset: NaN
}

template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void k_distill(DistillArgs a) {
    __shared__ uint32_t bits[NT * NV / 4];
    __shared__ Part sh_part[NT / 64];
    __shared__ Bulk sh_bulk;
    // a queue gives out the parts of every queues-th row, row by row: the parts of all but its last row
    // run, so no more than queues * (parts - 1) workgroups ever wait for one that has not begun
    Ticket at{0u, blockIdx.x};
    if (a.tickets) at = take_ticket(a.tickets, a.queues);
    const int64_t r = (int64_t)(at.number / (uint32_t)a.parts) * a.queues + at.queue;
    const int part = (int)(at.number % (uint32_t)a.parts), j0 = part * NT * NV;
    if (r >= a.n) return;
    const Row<T> row(a.x + r * a.ld_bytes, a.v);
    uint4 raw[NV];
    load_part<T, NT, NV>(row, j0, raw);
    const float c = kLog2e / a.temperature;
    const int col = column_of(a, r);
    mark_kept<NT, NV>(bits, col >= 0, col >= 0 ? row.vector_of(col) - j0 : -1, (col + row.head) % T::kVec);
    Kept k{-1, 0.0f, 0.0f};
    const bool finish = part == 0 && threadIdx.x < 64;
    if (finish) k = load_kept(a, r, col, row);
    Part p = block_merge<NT>(sum_part<T, NT, NV>(raw, c, a.rest, bits), c, sh_part);
    uint64_t* words = a.words + r * (a.parts + 2);
    if (a.tickets && threadIdx.x == 0) publish(words + part, word(p.m, p.s));
    float kept_grad = 0.0f;
    if (finish) {
        if (a.tickets) {
            p = no_part();
            for (int i = threadIdx.x; i < a.parts; i += 64) {
                const uint64_t w = wait_for(words + i);
                p = merge(p, Part{word_a(w), word_b(w), 0.0f}, c);
            }
            p = wave_merge(p, c);
        }
        const Bulk b = finish_row<T>(a, r, k, p, kept_grad);
        if (threadIdx.x == 0) {
            sh_bulk = b;
            if (a.tickets && a.out) {
                publish(words + a.parts, word(b.m, b.log2_s));
                publish(words + a.parts + 1, word(b.factor, 0.0f));
            }
        }
    }
    if (!a.out) return;
    if (part != 0 && threadIdx.x == 0) {
        const uint64_t w = wait_for(words + a.parts), f = wait_for(words + a.parts + 1);
        sh_bulk = Bulk{word_a(w), word_b(w), word_a(f)};
    }
    __syncthreads();
    const Writer w = writer_of(sh_bulk, c);
    char* out = a.out + r * a.out_ld_bytes;
    store_part<T, NT, NV>(
        row, out, j0,
        [&](int i, float (&f)[T::kVec]) {
            unpack(again(raw[i]), f, T());
            gradient(f, c, w);
        },
        [&](int i) { return (uint32_t)((const uint8_t*)bits)[i * NT + threadIdx.x]; });
    if (finish && k.col >= 0) T::store(out + k.col * T::kSize, kept_grad);
}

// ---- the loss alone -----------------------------------------------------------------------------------
// Nothing is to be written after the sums, so no part waits: a launch for the parts and one, a wave a
// row, that joins them.  1777 x 50021 float16: 38 + 5 us, 4.0 TB/s in all (with parts that wait 60 us).
template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void k_distill_parts(DistillArgs a) {
    __shared__ uint32_t bits[NT * NV / 4];
    __shared__ Part sh_part[NT / 64];
    const int64_t r = blockIdx.x / (uint32_t)a.parts;
    const int part = (int)(blockIdx.x % (uint32_t)a.parts), j0 = part * NT * NV;
    const Row<T> row(a.x + r * a.ld_bytes, a.v);
    uint4 raw[NV];
    load_part<T, NT, NV>(row, j0, raw);
    const float c = kLog2e / a.temperature;
    if (a.rest) {
        const int col = column_of(a, r);
        mark_kept<NT, NV>(bits, col >= 0, col >= 0 ? row.vector_of(col) - j0 : -1, (col + row.head) % T::kVec);
    }
    const Part p = block_merge<NT>(sum_part<T, NT, NV>(raw, c, a.rest, bits), c, sh_part);
    if (threadIdx.x == 0) a.words[blockIdx.x] = word(p.m, p.s);
}
template <typename T>
__global__ __launch_bounds__(64) void k_distill_join(DistillArgs a) {
    const int64_t r = blockIdx.x;
    const Row<T> row(a.x + r * a.ld_bytes, a.v);
    const Kept k = load_kept(a, r, column_of(a, r), row);
    const float c = kLog2e / a.temperature;
    Part p = no_part();
    for (int i = threadIdx.x; i < a.parts; i += 64) {
        const uint64_t w = a.words[r * a.parts + i];
        p = merge(p, Part{word_a(w), word_b(w), 0.0f}, c);
    }
    float none;
    finish_row<T>(a, r, k, wave_merge(p, c), none);
}

// A wave a row while the row fits its registers; 256 lanes and 8 vectors beyond, or fewer vectors
// while that leaves too few workgroups to fill 256 CUs.
inline Shape distill_shape(int64_t n, int64_t nvec) {
    Shape s{256, 8, 1, 1};
    if (nvec <= 64 * 8) {
        s.nt = 64;
        s.nv = nvec <= 64 ? 1 : nvec <= 128 ? 2 : nvec <= 256 ? 4 : 8;
    } else {
        while (s.nv > 1 && n * ceil_div(nvec, 256 * s.nv) < 1024 && ceil_div(nvec, 128 * s.nv) <= kMaxParts) s.nv /= 2;
    }
    s.parts = (int)ceil_div(nvec, (int64_t)s.nt * s.nv);
    return s;
}
inline int64_t distill_scratch(const Shape& s, int64_t n) { return s.parts == 1 ? 0 : kTicketBytes + 8 * n * (s.parts + 2); }

}  // namespace logits

int use_guard_distill(const uint32_t* looks, bool* gave_up) { return use_guard(looks, gave_up); }
}  // namespace ddm

using namespace ddm;
using namespace ddm::logits;

extern "C" int64_t ddm_topk_distill_scratch_bytes(int64_t n, int64_t v, int32_t dtype) {
    if (n <= 0 || v < 1 || v > kMaxColumns) return 0;
    const int vec = dtype == DDM_F32 ? 4 : 8;            // whether rows start aligned or not
    const int64_t a = distill_scratch(distill_shape(n, ceil_div(v, vec)), n);
    const int64_t b = distill_scratch(distill_shape(n, ceil_div(v + vec - 1, vec)), n);
    return a > b ? a : b;
}

extern "C" int ddm_topk_distill(const void* logits, int32_t dtype, int64_t n, int64_t v, int64_t ld, const void* index,
                                int32_t index_bytes, const float* logprob, int32_t k, int32_t tail, float temperature,
                                const float* weight, float* loss, void* grad, int64_t grad_ld, void* scratch,
                                ddm_stream_t stream, ddm_event_t ev_begin, ddm_event_t ev_end) {
    if (int rc = check_rows("ddm_topk_distill", dtype, n, v, ld, index_bytes, temperature, k)) return rc;
    if (tail != DDM_TAIL_RENORM && tail != DDM_TAIL_REST) {
        set_error("ddm_topk_distill: unknown tail %d", (int)tail);
        return DDM_E_ARG;
    }
    if (tail == DDM_TAIL_REST && temperature != 1.0f) {
        set_error("ddm_topk_distill: the remainder's probability is known at temperature 1 only");
        return DDM_E_ARG;
    }
    if (n == 0) return timed_nothing(ev_begin, ev_end, stream);
    const int size = dtype == DDM_F32 ? 4 : 2;
    const Shape s = distill_shape(n, vectors_of(logits, ld * size, v, 16 / size));
    if (int rc = check_grid("ddm_topk_distill", n * s.parts + kQueues * kDies * s.parts, s.nt)) return rc;
    if (!logits || !loss || (k && (!index || !logprob)) || (grad && grad_ld < v) || (s.parts > 1 && !scratch)) {
        set_error("ddm_topk_distill: invalid argument (null pointer or gradient stride)");
        return DDM_E_ARG;
    }
    const hipStream_t st = as_hip(stream);
    return timed(ev_begin, ev_end, st, [&] {
        return with_type(dtype, [&](auto type) {
            using T = decltype(type);
            DistillArgs a{(const char*)logits, n, v, ld * T::kSize, grad_ld * T::kSize, index, index_bytes == 8, logprob,
                          weight, k, tail == DDM_TAIL_REST, s.parts, temperature, loss, (char*)grad, nullptr, 1, nullptr};
            if (s.parts > 1 && !grad) {
                a.words = (uint64_t*)scratch;
                with_part_shape(s, [&](auto nt, auto nv) {
                    k_distill_parts<T, nt(), nv()><<<dim3((unsigned)(n * s.parts)), nt(), 0, st>>>(a);
                });
                if (int rc = launch_status("ddm_topk_distill")) return rc;
                k_distill_join<T><<<dim3((unsigned)n), 64, 0, st>>>(a);
                return launch_status("ddm_topk_distill");
            }
            if (s.parts > 1) {
                a.tickets = (uint32_t*)scratch;
                while (a.queues < kQueues && a.queues * 2 * s.parts <= 128) a.queues *= 2;
                a.words = (uint64_t*)((char*)scratch + kTicketBytes);
                if (int rc = reset_words(a.tickets, a.words, n * (s.parts + 2), nullptr, nullptr, 0, st, "ddm_topk_distill"))
                    return rc;
            }
            with_part_shape(s, [&](auto nt, auto nv) {
                k_distill<T, nt(), nv()><<<dim3((unsigned)(a.tickets ? queue_grid(ceil_div(n, a.queues) * s.parts, a.queues) : n * s.parts)), nt(), 0, st>>>(a);
            });
            return launch_status("ddm_topk_distill");
        });
    });
}
