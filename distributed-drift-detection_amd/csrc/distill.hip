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
// Bound by reading the logits once and writing the gradient once.  A row that fits one
// workgroup's registers (1024 lanes of 16 vectors: 131072 16-bit entries) is read once, summed
// while it arrives, and written from the registers; longer rows, and rows too few to fill the
// chip with a workgroup each, are cut into parts, summed, finished by a wave a row and written
// by a second reading.
#include "logits.h"

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
    float2* part_sum;          // [n][parts] m, s of what is not kept (renorm: of everything)
    float4* coef;              // [n] the bulk's m, log2 s and factor
    int32_t* kept;             // [n][k] column, or -1
    float* kept_grad;          // [n][k]
};

// The teacher's alternatives of a row, one a lane of a wave.
struct Kept {
    int col;                   // -1: none
    float l, x;                // teacher's log probability, student's logit
};

template <typename T>
__device__ __forceinline__ Kept load_kept(const DistillArgs& a, int64_t r, const Row<T>& row) {
    const int lane = threadIdx.x & 63;
    Kept k{-1, -INFINITY, -INFINITY};
    if (lane < a.k) {
        const int64_t c = target_at(a.index, a.index_wide, r * a.k + lane);
        k.col = c >= 0 && c < a.v ? (int)c : -1;
        k.l = a.logprob[r * a.k + lane];
    }
    for (int j = 0; j + 1 < a.k; ++j)                    // the first of equal columns counts
        if (lane > j && k.col == __builtin_amdgcn_readlane(k.col, j)) k.col = -1;
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

template <typename T>
__device__ __forceinline__ void write_vector(const Row<T>& row, char* out, int j, const uint4& raw, float c,
                                             const Bulk& b) {
    float f[T::kVec];
    unpack(raw, f, T());
#pragma unroll
    for (int e = 0; e < T::kVec; ++e)
        f[e] = b.factor == 0.0f ? 0.0f : __builtin_amdgcn_exp2f((f[e] - b.m) * c - b.log2_s) * b.factor;
    row.store(out, j, f);
}

// ---- a row in one workgroup's registers -------------------------------------------------------------
template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void k_distill_rows(DistillArgs a) {
    __shared__ uint32_t bits[NT * NV / 4];
    __shared__ Part sh_part[NT / 64];
    __shared__ Bulk sh_bulk;
    const int64_t r = blockIdx.x;
    const Row<T> row(a.x + r * a.ld_bytes, a.v);
    uint4 raw[NV];
    load_part<T, NT, NV>(row, 0, raw);
    const float c = kLog2e / a.temperature;
    Kept k{-1, 0.0f, 0.0f};
    if (threadIdx.x < 64) k = load_kept(a, r, row);
    if (a.rest) mark_kept<NT, NV>(bits, k.col >= 0, row.vector_of(k.col), (k.col + row.head) % T::kVec);
    const Part p = block_merge<NT>(sum_part<T, NT, NV>(raw, c, a.rest, bits), c, sh_part);
    float kept_grad = 0.0f;
    if (threadIdx.x < 64) {
        const Bulk b = finish_row<T>(a, r, k, p, kept_grad);
        if (threadIdx.x == 0) sh_bulk = b;
    }
    if (!a.out) return;
    __syncthreads();
    const Bulk b = sh_bulk;
    char* out = a.out + r * a.out_ld_bytes;
#pragma unroll
    for (int i = 0; i < NV; ++i) write_vector(row, out, i * NT + (int)threadIdx.x, again(raw[i]), c, b);
    __syncthreads();
    if (threadIdx.x < 64 && k.col >= 0) T::store(out + k.col * T::kSize, kept_grad);
}

// ---- rows in parts ------------------------------------------------------------------------------------
template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void k_distill_parts(DistillArgs a) {
    __shared__ uint32_t bits[NT * NV / 4];
    __shared__ Part sh_part[NT / 64];
    const int64_t r = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x % a.parts), j0 = part * NT * NV;
    const Row<T> row(a.x + r * a.ld_bytes, a.v);
    uint4 raw[NV];
    load_part<T, NT, NV>(row, j0, raw);
    const float c = kLog2e / a.temperature;
    if (a.rest) {                                       // repeats set the same bit twice
        int64_t col = -1;
        if (threadIdx.x < a.k) col = target_at(a.index, a.index_wide, r * a.k + threadIdx.x);
        const bool in = col >= 0 && col < a.v;
        mark_kept<NT, NV>(bits, in, in ? row.vector_of((int)col) - j0 : -1, in ? ((int)col + row.head) % T::kVec : 0);
    }
    const Part p = block_merge<NT>(sum_part<T, NT, NV>(raw, c, a.rest, bits), c, sh_part);
    if (threadIdx.x == 0) a.part_sum[r * a.parts + part] = make_float2(p.m, p.s);
}

template <typename T>
__global__ __launch_bounds__(64) void k_distill_join(DistillArgs a) {
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x;
    const Row<T> row(a.x + r * a.ld_bytes, a.v);
    const Kept k = load_kept(a, r, row);
    Part p = no_part();
    if (lane < a.parts) {
        const float2 q = a.part_sum[r * a.parts + lane];
        p.m = q.x;
        p.s = q.y;
    }
    p = wave_merge(p, kLog2e / a.temperature);
    float kept_grad;
    const Bulk b = finish_row<T>(a, r, k, p, kept_grad);
    if (!a.out) return;
    if (lane == 0) a.coef[r] = make_float4(b.m, b.log2_s, b.factor, 0.0f);
    if (lane < a.k) {
        a.kept[r * a.k + lane] = k.col;
        a.kept_grad[r * a.k + lane] = kept_grad;
    }
}

template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void k_distill_grad(DistillArgs a) {
    const int64_t r = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x % a.parts), j0 = part * NT * NV;
    const Row<T> row(a.x + r * a.ld_bytes, a.v);
    uint4 raw[NV];
    load_part<T, NT, NV>(row, j0, raw);
    const float4 q = a.coef[r];
    const Bulk b{q.x, q.y, q.z};
    const float c = kLog2e / a.temperature;
    char* out = a.out + r * a.out_ld_bytes;
#pragma unroll
    for (int i = 0; i < NV; ++i) write_vector(row, out, j0 + i * NT + (int)threadIdx.x, raw[i], c, b);
    __syncthreads();
    if (threadIdx.x < a.k) {
        const int col = a.kept[r * a.k + threadIdx.x];
        const int j = col >= 0 ? row.vector_of(col) - j0 : -1;
        if (j >= 0 && j < NT * NV) T::store(out + col * T::kSize, a.kept_grad[r * a.k + threadIdx.x]);
    }
}

// A workgroup a row while it fits and there are rows enough to give every CU one or two, or
// nothing is gained by cutting it; parts as for the scores otherwise.
inline Shape distill_shape(int64_t n, int64_t nvec, bool grad) {
    Shape s{256, 8, 1, 1};
    if (nvec <= 64 * 8) {
        s.nt = 64;
        s.nv = nvec <= 64 ? 1 : nvec <= 128 ? 2 : nvec <= 256 ? 4 : 8;
    } else if (grad && n >= 256 && nvec <= 1024 * 16) {
        s.nt = nvec <= 256 * 8 ? 256 : 1024;
        s.nv = nvec <= 256 * 4 ? 4 : nvec <= 256 * 8 ? 8 : nvec <= 1024 * 4 ? 4 : nvec <= 1024 * 8 ? 8 : 16;
    } else {
        while (s.nv > 1 && n * ceil_div(nvec, 256 * s.nv) < 1024 && ceil_div(nvec, 128 * s.nv) <= kMaxParts) s.nv /= 2;
    }
    s.parts = (int)ceil_div(nvec, (int64_t)s.nt * s.nv);
    return s;
}
inline int64_t distill_scratch(const Shape& s, int64_t n, int64_t k) {
    return s.parts == 1 ? 0 : n * (16 + 8 * (int64_t)s.parts + 8 * k);
}

}  // namespace logits
}  // namespace ddm

using namespace ddm;
using namespace ddm::logits;

extern "C" int64_t ddm_topk_distill_scratch_bytes(int64_t n, int64_t v, int32_t dtype, int32_t k, int32_t grad) {
    if (n <= 0 || v < 1 || v > kMaxColumns || k < 0 || k > kMaxTop) return 0;
    const int vec = dtype == DDM_F32 ? 4 : 8;            // whether rows start aligned or not
    const int64_t a = distill_scratch(distill_shape(n, ceil_div(v, vec), grad != 0), n, k);
    const int64_t b = distill_scratch(distill_shape(n, ceil_div(v + vec - 1, vec), grad != 0), n, k);
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
    if (n == 0) return 0;
    const int size = dtype == DDM_F32 ? 4 : 2;
    const Shape s = distill_shape(n, vectors_of(logits, ld * size, v, 16 / size), grad != nullptr);
    if (!logits || !loss || (k && (!index || !logprob)) || (grad && grad_ld < v) || (s.parts > 1 && !scratch)) {
        set_error("ddm_topk_distill: invalid argument (null pointer or gradient stride)");
        return DDM_E_ARG;
    }
    const hipStream_t st = as_hip(stream);
    return timed(ev_begin, ev_end, st, [&] {
        return with_type(dtype, [&](auto type) {
            using T = decltype(type);
            char* w = (char*)scratch;
            DistillArgs a{(const char*)logits, n, v, ld * T::kSize, grad_ld * T::kSize, index, index_bytes == 8, logprob,
                          weight, k, tail == DDM_TAIL_REST, s.parts, temperature, loss, (char*)grad,
                          (float2*)(w + n * 16), (float4*)w, (int32_t*)(w + n * (16 + 8 * (int64_t)s.parts)),
                          (float*)(w + n * (16 + 8 * (int64_t)s.parts + 4 * (int64_t)k))};
            if (s.parts == 1) {
                with_row_shape(s, [&](auto nt, auto nv) { k_distill_rows<T, nt(), nv()><<<dim3((unsigned)n), nt(), 0, st>>>(a); });
                return launch_status("ddm_topk_distill");
            }
            const dim3 grid((unsigned)(n * s.parts));
            auto each_part = [&](auto launch) {
                if (s.nv == 1) launch(std::integral_constant<int, 1>());
                if (s.nv == 2) launch(std::integral_constant<int, 2>());
                if (s.nv == 4) launch(std::integral_constant<int, 4>());
                if (s.nv == 8) launch(std::integral_constant<int, 8>());
            };
            each_part([&](auto nv) { k_distill_parts<T, 256, nv()><<<grid, 256, 0, st>>>(a); });
            if (int rc = launch_status("ddm_topk_distill")) return rc;
            k_distill_join<T><<<dim3((unsigned)n), 64, 0, st>>>(a);
            if (int rc = launch_status("ddm_topk_distill")) return rc;
            if (grad) each_part([&](auto nv) { k_distill_grad<T, 256, nv()><<<grid, 256, 0, st>>>(a); });
            return launch_status("ddm_topk_distill");
        });
    });
}
