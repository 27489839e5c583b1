// Gated linear recurrence over ragged sequences, its gradient and its single step:
//   a_t = exp(l_t),  b_t = x_t | (1 - a_t) x_t | sqrt(1 - a_t^2) x_t,  h_t = a_t h_{t-1} + b_t,
// per channel, from a carried state, back into it.  With the second form it is the
// exponentially weighted chart of a stream of scores; the others are a recurrent layer's.
//
// A composition of steps is a step: (A1, B1) then (A2, B2) is (A1 A2, A2 B1 + B2).  Rows are cut
// into tiles; a workgroup holds one tile of rows and channels in registers, reduces it to
// its (A, B), gets the state before it from the tiles before it, and runs the recurrence from
// there: x and l are read once and h is written once, which is the floor.  The state comes
// by a look-back of fixed shape: tiles form groups, a tile reads the (A, B) of those before it in
// its group and the state after the group before, which that group's last tile publishes.
// What is composed in which order depends on the sizes alone, so results do not change from
// run to run.  Tiles are taken in order by a ticket, so that a tile only ever waits for tiles
// that already run.  A published word is one 8-byte store that carries its own validity (unset
// words hold all ones), so no fence is needed.
//
// Sequences need no alignment with tiles: at a sequence's first row the state before it is cut
// off, (A, B) = (cut, a state + b), and the cut is a mark of its own (A < 0) rather than a zero
// factor, so that what one sequence overflows or poisons does not reach the next.
//
// The gradient is the same recurrence backwards: u_t = a_t g_t with g_t = dh_t + u_{t+1} (at a
// last row dh_t + dstate), dx = g db/dx, dl = g (a h_{t-1} + db/dl), dstate_in = u at the first row.
// The gradient of a gate that several channels share is summed in a fixed tree over their lanes,
// and over the rest in a second launch.
#pragma once
#include <initializer_list>
#include <type_traits>

#include "common.h"

namespace ddm {
namespace gated {

constexpr int NT = 512, W = NT / 64;
constexpr uint64_t kUnset = ~0ull;
constexpr uint32_t kSpinLimit = 1u << 22;      // a tile's predecessors run already: a guard, not a wait
constexpr float kCut = -1.0f;                   // A of a step that forgets what was before it

template <typename E_, int CODE>
struct type_of {
    typedef E_ E;
    static constexpr int kCode = CODE;
};
typedef type_of<float, DDM_F32> f32_t;
typedef type_of<__bf16, DDM_BF16> bf16_t;
typedef type_of<_Float16, DDM_F16> f16_t;

template <typename T, int N>
struct alignas(sizeof(typename T::E) * N) Raw {
    typename T::E e[N];
};

struct Args {
    const char *x, *l, *h, *dh;          // dh: the gradient's only; h: forward's output, its input
    char *out, *dx, *dl;
    int64_t ld_x, ld_l, ld_h, ld_dh, ld_dx, ld_dl;      // bytes a row
    int64_t rows;
    int d, share, scale, fill;           // share: channels a gate
    const int64_t* off;                   // NULL: one sequence of all rows
    int64_t n;
    const float *state_in, *dstate;      // may be NULL (0)
    float* state_out;                     // state after, or gradient of the state before
    int cl_bits, ncb, group;             // lanes across channels (log2), channel blocks, tiles a group
    int64_t ntiles;
    uint32_t* ticket;                     // NULL: one tile, no chain
    uint64_t *agg, *inc;                  // [ntiles][dp], [groups][dp]
    int64_t dp;
    float* dl_part;                       // [rows][parts a row] or NULL: dl itself
    int dl_width;                         // lanes summed within a wave
};

struct Step {
    float a, b;
};
__device__ __forceinline__ Step after(const Step& p, const Step& q) {   // p, then q
    Step r;
    r.a = q.a < 0.0f ? kCut : p.a < 0.0f ? (q.a != q.a ? q.a : kCut) : p.a * q.a;
    r.b = q.a < 0.0f ? q.b : fmaf(q.a, p.b, q.b);
    return r;
}
__device__ __forceinline__ float apply(const Step& s, float h) { return s.a < 0.0f ? s.b : fmaf(s.a, h, s.b); }

// ---- gates ---------------------------------------------------------------------------------------
// 1 - e^y without cancellation: a series up to |y| = 0.7 (the first term left out is under 2^-27 of
// the result), the difference beyond, where e^y is at most half.
__device__ __forceinline__ float one_minus_exp(float y) {
    float p = 2.7557319e-7f;                        // 1/10!
    p = fmaf(p, y, 2.7557319e-6f);
    p = fmaf(p, y, 2.4801587e-5f);
    p = fmaf(p, y, 1.9841270e-4f);
    p = fmaf(p, y, 1.3888889e-3f);
    p = fmaf(p, y, 8.3333333e-3f);
    p = fmaf(p, y, 4.1666667e-2f);
    p = fmaf(p, y, 1.6666667e-1f);
    p = fmaf(p, y, 0.5f);
    p = fmaf(p, y, 1.0f);
    return fabsf(y) <= 0.7f ? -y * p : 1.0f - __builtin_amdgcn_exp2f(y * 1.4426950408889634f);
}
// e^l: the product's rounding, carried, keeps the exponential's error at its own.
__device__ __forceinline__ float gate(float l) {
    const float y = l * 1.4426950408889634f;
    const float r = fmaf(l, 1.4426950408889634f, -y);
    const float e = __builtin_amdgcn_exp2f(y);
    return fabsf(y) < 126.0f ? fmaf(e * 0.6931471805599453f, r, e) : e;
}
__device__ __forceinline__ float input_factor(float l, int scale) {
    if (scale == DDM_GATED_NONE) return 1.0f;
    if (scale == DDM_GATED_EWMA) return one_minus_exp(l);
    return __builtin_amdgcn_sqrtf(fmaxf(one_minus_exp(2.0f * l), 0.0f));
}
// ... and its derivative by l.
__device__ __forceinline__ float input_slope(float a, float f, int scale) {
    if (scale == DDM_GATED_NONE) return 0.0f;
    if (scale == DDM_GATED_EWMA) return -a;
    return f > 0.0f ? -(a * a) / f : f - f;        // NaN stays NaN
}

// ---- a tile's place -------------------------------------------------------------------------------
struct Place {
    int64_t tile;          // in the order of the recurrence
    int block;             // of channels
};
__device__ __forceinline__ Place take(const Args& a) {
    __shared__ uint32_t sh;
    uint32_t t = blockIdx.x;
    if (a.ticket) {
        if (threadIdx.x == 0) sh = atomicAdd(a.ticket, 1u);
        __syncthreads();
        t = sh;
    }
    return Place{(int64_t)(t / (uint32_t)a.ncb), (int)(t % (uint32_t)a.ncb)};
}

// Which rows of [row0, row0 + nrows) begin and end a sequence (its number, or -1).
__device__ __forceinline__ void mark_rows(const Args& a, int64_t row0, int nrows, int32_t* begins, int32_t* ends) {
    for (int i = threadIdx.x; i < nrows; i += NT) begins[i] = ends[i] = -1;
    int64_t lo = 0, hi = a.n;                       // the first sequence that ends behind row0
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (a.off[mid + 1] > row0)
            hi = mid;
        else
            lo = mid + 1;
    }
    __syncthreads();
    for (int64_t s = lo + threadIdx.x; s < a.n; s += NT) {
        const int64_t b = a.off[s], e = a.off[s + 1];
        if (b >= row0 + nrows) break;
        if (e <= b) continue;
        if (b >= row0) begins[b - row0] = (int32_t)s;
        if (e > row0 && e <= row0 + nrows) ends[e - 1 - row0] = (int32_t)s;
    }
    __syncthreads();
}

// ---- the state before a lane's rows -----------------------------------------------------------------
template <int VEC>
struct ScanLds {
    float a[W][64 * VEC], b[W][64 * VEC];
};

// Steps of the workgroup's time groups composed in order, a channel apart: what is before the
// lane's own, and all together.
template <int VEC>
__device__ __forceinline__ void block_scan(const Step (&own)[VEC], int cl, ScanLds<VEC>& l, Step (&before)[VEC],
                                           Step (&all)[VEC]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Step s[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) s[v] = own[v];
    for (int d = cl; d < 64; d <<= 1) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Step p{__shfl_up(s[v].a, d), __shfl_up(s[v].b, d)};
            if (lane >= d) s[v] = after(p, s[v]);
        }
    }
    if (lane >= 64 - cl) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            l.a[wave][(lane & (cl - 1)) * VEC + v] = s[v].a;
            l.b[wave][(lane & (cl - 1)) * VEC + v] = s[v].b;
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        s[v] = Step{__shfl_up(s[v].a, cl), __shfl_up(s[v].b, cl)};
        if (lane < cl) s[v] = Step{1.0f, 0.0f};
        all[v] = Step{1.0f, 0.0f};
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (w == wave) before[v] = after(all[v], s[v]);
            const int c = (lane & (cl - 1)) * VEC + v;
            all[v] = after(all[v], Step{l.a[w][c], l.b[w][c]});
        }
    }
    __syncthreads();
}

__device__ __forceinline__ uint64_t pack(float a, float b) {
    const uint64_t w = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
    return w == kUnset ? w ^ 1u : w;               // two NaN of all ones: another NaN
}
__device__ __forceinline__ void publish(uint64_t* p, uint64_t w) {
    __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int N>
__device__ __forceinline__ void await(const uint64_t* p, uint64_t (&w)[N]) {
    for (uint32_t spin = 0;; ++spin) {
        bool set = true;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[i] = __hip_atomic_load(p + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            set = set && w[i] != kUnset;
        }
        if (set || spin == kSpinLimit) return;      // unset words are NaN
        __builtin_amdgcn_s_sleep(1);
    }
}

// From the steps of every lane's rows to the state before them.
template <int VEC>
__device__ __forceinline__ void chain(const Args& a, const Place& at, const Step (&own)[VEC], ScanLds<VEC>& l,
                                      float (&h)[VEC]) {
    const int cl = 1 << a.cl_bits, tg = threadIdx.x >> a.cl_bits;
    Step before[VEC], all[VEC];
    block_scan<VEC>(own, cl, l, before, all);
    float carry[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = 0.0f;
    if (a.ticket) {
        const int64_t c = ((int64_t)at.block * cl + (threadIdx.x & (cl - 1))) * VEC;
        const int64_t g = at.tile / a.group;
        const int in_group = (int)(at.tile % a.group);
        const bool last = in_group == a.group - 1;
        if (tg == 0 && !last && at.tile + 1 < a.ntiles) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) publish(a.agg + at.tile * a.dp + c + v, pack(all[v].a, all[v].b));
        }
        if (at.tile > 0) {
            // time groups share the tiles before this one in the group; the first also takes the
            // state before the group, a step that forgets everything
            Step p[VEC], none[VEC], sum[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) p[v] = Step{1.0f, 0.0f};
            uint64_t w[VEC];
            if (tg == 0 && g > 0) {
                await<VEC>(a.inc + (g - 1) * a.dp + c, w);
#pragma unroll
                for (int v = 0; v < VEC; ++v) p[v] = Step{kCut, __uint_as_float((uint32_t)w[v])};
            }
            const int per = (a.group + (NT >> a.cl_bits) - 1) / (NT >> a.cl_bits);
            for (int i = 0; i < per; ++i) {
                const int j = tg * per + i;
                if (j < in_group) {
                    await<VEC>(a.agg + (g * a.group + j) * a.dp + c, w);
#pragma unroll
                    for (int v = 0; v < VEC; ++v)
                        p[v] = after(p[v], Step{__uint_as_float((uint32_t)w[v]), __uint_as_float((uint32_t)(w[v] >> 32))});
                }
            }
            block_scan<VEC>(p, cl, l, none, sum);
#pragma unroll
            for (int v = 0; v < VEC; ++v) carry[v] = apply(sum[v], 0.0f);
        }
        if (tg == 0 && last && at.tile + 1 < a.ntiles) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) publish(a.inc + g * a.dp + c + v, pack(apply(all[v], carry[v]), 0.0f));
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = apply(before[v], carry[v]);
}

template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> load(const char* base, int64_t ld, int64_t row, int c) {
    return *(const Raw<T, VEC>*)(base + row * ld + (int64_t)c * sizeof(typename T::E));
}
template <typename T, int VEC>
__device__ __forceinline__ void store(char* base, int64_t ld, int64_t row, int c, const float (&f)[VEC]) {
    Raw<T, VEC> r;
#pragma unroll
    for (int v = 0; v < VEC; ++v) r.e[v] = (typename T::E)f[v];
    *(Raw<T, VEC>*)(base + row * ld + (int64_t)c * sizeof(typename T::E)) = r;
}
// The gates of VEC channels: their own, or one that they share.
template <typename L, int VEC, bool OWN>
struct Gates {
    Raw<L, OWN ? VEC : 1> r;
    __device__ __forceinline__ void load_row(const Args& a, int64_t row, int c) {
        r = load<L, OWN ? VEC : 1>(a.l, a.ld_l, row, OWN ? c : c / a.share);
    }
    __device__ __forceinline__ float operator[](int v) const { return (float)r.e[OWN ? v : 0]; }
};

// ---- launch shapes ---------------------------------------------------------------------------------
struct Shape {
    int vec, cl_bits, ncb, r, group, dl_width, dl_parts;
    int64_t ntiles, dp;
    int64_t words() const { return ntiles > 1 ? (ntiles + ceil_div(ntiles, group)) * dp : 0; }
};
inline Shape shape_of(int64_t rows, int d, int share, int vec, bool grad) {
    Shape s;
    s.vec = vec;
    const int lanes = d / vec;
    s.cl_bits = 0;
    while ((1 << s.cl_bits) < lanes && s.cl_bits < 6) ++s.cl_bits;
    s.ncb = (int)ceil_div(lanes, 1 << s.cl_bits);
    const int tg = NT >> s.cl_bits;
    // rows a lane: many, so that a tile's share of the chain is small, unless that leaves CUs idle
    // or makes a tile's marks outgrow 16 KB of LDS
    s.r = grad ? 8 : 16;
    if (ceil_div(rows, tg * s.r) * s.ncb < 512 || tg * s.r > 2048) s.r = grad ? 2 : 4;
    s.ntiles = ceil_div(rows, (int64_t)tg * s.r);
    s.group = tg * 2 < 64 ? tg * 2 : 64;
    s.dp = (int64_t)(s.ncb << s.cl_bits) * vec;
    s.dl_width = 1;
    s.dl_parts = 0;
    if (grad && share > 1) {
        int units = share / vec;
        while (units % 2 == 0 && s.dl_width < (1 << s.cl_bits)) {
            units /= 2;
            s.dl_width *= 2;
        }
        s.dl_parts = units > 1 ? units : 0;
    }
    return s;
}

inline int elem_size(int32_t dtype) { return dtype == DDM_F32 ? 4 : 2; }
inline int wide_vec(int32_t dtype) { return 8 / elem_size(dtype); }

// 8 bytes of x a lane where every operand's rows are aligned for it and no such piece has two
// gates; else an entry a lane.
inline int vec_of(int32_t dtype, int32_t gate_dtype, int d, int share, std::initializer_list<const void*> x,
                  std::initializer_list<int64_t> ld, const void* l, int64_t ld_l, const void* dl, int64_t ld_dl) {
    const int v = wide_vec(dtype), es = elem_size(dtype), gs = elem_size(gate_dtype);
    if (d % v || (share > 1 && share % v)) return 1;
    for (const void* p : x)
        if ((uintptr_t)p % 8) return 1;
    for (int64_t s : ld)
        if (s * es % 8) return 1;
    if (share == 1 && ((uintptr_t)l % (v * gs) || ld_l * gs % (v * gs) || (uintptr_t)dl % (v * gs) || ld_dl * gs % (v * gs)))
        return 1;
    return v;
}

template <typename F>
int with_types(int32_t dtype, int32_t gate_dtype, F f) {
    if (dtype == DDM_F32) return f(f32_t(), f32_t());
    if (dtype == DDM_BF16) return gate_dtype == DDM_F32 ? f(bf16_t(), f32_t()) : f(bf16_t(), bf16_t());
    return gate_dtype == DDM_F32 ? f(f16_t(), f32_t()) : f(f16_t(), f16_t());
}
template <typename F>
void with_vec(int vec, bool own, F f) {
    if (vec == 1) {
        if (own) return f(std::integral_constant<int, 1>(), std::true_type());
        return f(std::integral_constant<int, 1>(), std::false_type());
    }
    if (own) return f(std::integral_constant<int, 0>(), std::true_type());     // 0: the type's wide one
    return f(std::integral_constant<int, 0>(), std::false_type());
}

inline int check(const char* who, int32_t dtype, int32_t gate_dtype, int64_t rows, int64_t d, int64_t gates,
                 int64_t ld_x, int64_t ld_l, int64_t n, int32_t scale) {
    if ((dtype != DDM_F32 && dtype != DDM_BF16 && dtype != DDM_F16) || (gate_dtype != dtype && gate_dtype != DDM_F32)) {
        set_error("%s: types %d and %d (gates of the inputs' type, or float32)", who, (int)dtype, (int)gate_dtype);
    } else if (rows < 0 || d < 1 || d > 1 << 20 || gates < 1 || d % gates || ld_x < d || (ld_l < gates && ld_l != 0) ||
               rows > (int64_t)1 << 40 || n < 0 || n > INT32_MAX) {
        set_error("%s: invalid argument (rows %lld, channels %lld, gates %lld that divide them, strides %lld and %lld)",
                  who, (long long)rows, (long long)d, (long long)gates, (long long)ld_x, (long long)ld_l);
    } else if (scale != DDM_GATED_NONE && scale != DDM_GATED_EWMA && scale != DDM_GATED_UNIT) {
        set_error("%s: unknown scale %d", who, (int)scale);
    } else {
        return 0;
    }
    return DDM_E_ARG;
}

// 0, or DDM_E_ARG where the grid has no room for the tiles.
inline int check_grid(const char* who, const Shape& s) {
    if (s.ntiles * s.ncb <= INT32_MAX) return 0;
    set_error("%s: %lld tiles of %d channel blocks", who, (long long)s.ntiles, s.ncb);
    return DDM_E_ARG;
}

inline int64_t scratch_bytes(const Shape& s, int64_t rows, int d) {
    const int64_t parts = s.dl_parts ? rows * (d / (s.vec * s.dl_width)) : 0;
    return (s.words() ? 16 + 8 * s.words() : 0) + 4 * parts;
}

// The chain's buffers and the copy of the states, with their launch where either is needed (gated.hip).
int begin(Args& a, const Shape& s, void* scratch, const float* from, float* to, int64_t nstate, hipStream_t st);

}  // namespace gated
}  // namespace ddm
