// Gated linear recurrence over ragged sequences, its gradient and its single step:
//   a_t = exp(l_t),  b_t = x_t | (1 - a_t) x_t | sqrt(1 - a_t^2) x_t,  h_t = a_t h_{t-1} + b_t,
// per channel, from a carried state, back into it.  With the second form it is the
// exponentially weighted chart of a stream of scores; the others are a recurrent layer's.
//
// A composition of steps is a step: (A1, B1) then (A2, B2) is (A1 A2, A2 B1 + B2).  Rows are cut
// into tiles; a workgroup holds one tile of rows and channels in registers, reduces it to
// its (A, B), gets the state before it from the tiles before it, and runs the recurrence from
// there: x and l are read once and h is written once, which is the floor.  The state comes
// by a look-back of fixed shape: tiles form groups and groups form rows of groups; a tile reads the
// (A, B) of those before it in its group, of the groups before that one in its row, which a group's
// last tile publishes, and the state after the row before.
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

#include "words.h"

namespace ddm {
namespace gated {

constexpr int NT = 512, W = NT / 64;
constexpr float kCut = -1.0f;                   // A of a step that forgets what was before it

template <typename E_, int CODE>
struct type_of {
    typedef E_ E;
    static constexpr int kCode = CODE;
};
typedef type_of<float, DDM_F32> f32_t;
typedef type_of<__bf16, DDM_BF16> bf16_t;
typedef type_of<_Float16, DDM_F16> f16_t;

// N entries of a row in as few registers as they have words; unpacked where they are used.
template <typename T, int N>
struct Raw {
    static constexpr int kBytes = (int)sizeof(typename T::E) * N, kWords = (kBytes + 3) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const char* p) {
        if (kBytes == 2)
            w[0] = *(const uint16_t*)p;
        else if (kBytes == 4)
            w[0] = *(const uint32_t*)p;
        else
            *(uint2*)w = *(const uint2*)p;
    }
    __device__ __forceinline__ float operator[](int i) const {
        if (sizeof(typename T::E) == 4) return __uint_as_float(w[i]);
        if (std::is_same<typename T::E, __bf16>::value) return __uint_as_float(i ? w[0] & 0xffff0000u : w[0] << 16);
        const uint16_t h = (uint16_t)(i ? w[0] >> 16 : w[0]);
        _Float16 f;
        __builtin_memcpy(&f, &h, 2);
        return (float)f;
    }
    // What was computed from it is not worth registers until it is used again.
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
    }
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
    int cl_bits, ncb, group;             // lanes across channels (log2), channel blocks, tiles a group and groups a row
    int64_t ntiles;
    uint32_t *tickets, queues;            // NULL: one tile, no chain
    uint64_t *agg, *inc, *far;            // [ntiles][dp], [groups][dp], [rows of groups][dp]
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
// 1 - e^y without cancellation, given e = e^y: for |y| <= 0.5 by (e^y - 1) / y, interpolated there in
// seven Chebyshev points (within 1.7 * 2^-24 of the value, 1.26 units in its last place, rounding included; over
// all float32 of [2^-6, 0.5]), beyond as the difference, where e is under 0.61.
__device__ __forceinline__ float one_minus_exp(float y, float e) {
    float p = 1.996217616e-4f;
    p = fmaf(p, y, 1.399777364e-3f);
    p = fmaf(p, y, 8.333181962e-3f);
    p = fmaf(p, y, 4.166530445e-2f);
    p = fmaf(p, y, 1.666666716e-1f);
    p = fmaf(p, y, 0.5000000596f);
    p = fmaf(p, y, 1.0f);
    return fabsf(y) <= 0.5f ? -y * p : 1.0f - e;
}
// a = e^l and the input's factor.  The exponential's argument is rounded once: half a step for each
// binary order that a loses, which is less the less a weighs.
struct Gate {
    float a, f;
};
template <int SCALE>
__device__ __forceinline__ Gate gate_of(float l) {
    Gate g;
    g.a = __builtin_amdgcn_exp2f(l * 1.4426950408889634f);
    g.f = SCALE == DDM_GATED_NONE ? 1.0f : one_minus_exp(l, g.a);
    if (SCALE == DDM_GATED_UNIT) {
        const float y = fmaf(g.f, g.a, g.f);                    // (1 - a)(1 + a)
        g.f = __builtin_amdgcn_sqrtf(y < 0.0f ? 0.0f : y);      // a NaN gate's stays NaN (a maximum would drop it)
    }
    return g;
}
// Gates are at most 1: products of theirs, which tiles and groups compose before they know the state, then
// cannot overflow where the recurrence itself would not.  One over 1 counts as NaN, so that what it reaches
// shows it.  (The scan asks first whether a wave has any: a select an entry took float32 scans
// from three workgroups a CU to two, and others spilled.)
template <int SCALE>
__device__ __forceinline__ Gate bounded_gate_of(float l) {
    Gate g = gate_of<SCALE>(l);
    if (g.a > 1.0f) {
        g.a = __builtin_nanf("");
        if (SCALE != DDM_GATED_NONE) g.f = g.a;
    }
    return g;
}
// The factor's derivative by l.
template <int SCALE>
__device__ __forceinline__ float slope_of(const Gate& g) {
    if (SCALE == DDM_GATED_NONE) return 0.0f;
    if (SCALE == DDM_GATED_EWMA) return -g.a;
    // a^2 / f by the reciprocal of 1 step's error
    return g.f > 0.0f ? -(g.a * g.a) * __builtin_amdgcn_rcpf(g.f) : g.f - g.f;        // NaN stays NaN
}
// f(std::integral_constant<int, scale>()): one branch a tile, not one an entry.
template <typename F>
__device__ __forceinline__ void with_scale(int scale, F f) {
    if (scale == DDM_GATED_NONE)
        f(std::integral_constant<int, DDM_GATED_NONE>());
    else if (scale == DDM_GATED_EWMA)
        f(std::integral_constant<int, DDM_GATED_EWMA>());
    else
        f(std::integral_constant<int, DDM_GATED_UNIT>());
}

// ---- a tile's place -------------------------------------------------------------------------------
struct Place {
    int64_t tile;          // in the order of the recurrence; from ntiles on: none
    int block;             // of channels
};
__device__ __forceinline__ Place take(const Args& a) {
    if (!a.tickets) return Place{0, (int)blockIdx.x};      // one tile
    // a queue gives out all tiles of every queues-th channel block, tile by tile
    const Ticket t = take_ticket(a.tickets, a.queues);
    // (the division is the vector unit's; its result is the same in every lane)
    const uint32_t blocks = (uint32_t)a.ncb / a.queues, tile = __builtin_amdgcn_readfirstlane(t.number / blocks);
    return Place{(int64_t)tile, (int)((t.number - tile * blocks) * a.queues + t.queue)};
}

// Which rows of a tile begin and end a sequence: a bit a row, and the sequence's number where it is set.
struct Marks {
    uint32_t *begin_bits, *end_bits;
    int32_t *begins, *ends;
    __device__ __forceinline__ Marks(int32_t* lds, int rows)
        : begin_bits((uint32_t*)lds), end_bits((uint32_t*)lds + rows / 32), begins(lds + rows / 16),
          ends(lds + rows / 16 + rows) {}
    static constexpr int bytes(int rows) { return (rows / 16 + 2 * rows) * 4; }
    // The lane's R rows from `at` on.
    template <int R>
    static __device__ __forceinline__ uint32_t lane(const uint32_t* bits, int at) {
        return (bits[at >> 5] >> (at & 31)) & ((1u << R) - 1u);
    }
};
// The sequences that may begin or end in a tile, one a thread, asked for before the tile's rows are, so
// that nobody waits for them behind those (65536 x 2048 in 37 sequences: 242 -> 220 us).
struct Sequences {
    int64_t s, b, e, first, end;       // a thread's first one; where the first begins and the last ends
};
__device__ __forceinline__ Sequences find_sequences(const Args& a, int64_t row0) {
    int64_t lo = 0, hi = a.n;
    // more than threads: the first that ends behind row0, in two rounds of loads for up to 4096: every
    // lane looks at the last of its 64th of what is left
    while (a.n > NT && lo < hi) {
        const int64_t step = (hi - lo + 63) / 64, i = lo + ((int64_t)(threadIdx.x & 63) + 1) * step - 1;
        const int before = __popcll(__ballot(i < hi && a.off[i + 1] <= row0));     // lanes wholly before
        lo += before * step;
        if (step == 1) break;
        hi = lo + step < hi ? lo + step : hi;
    }
    if (lo > a.n) lo = a.n;
    Sequences q{lo + threadIdx.x, 0, 0, a.off[0], a.off[a.n]};
    if (q.s < a.n) {
        q.b = a.off[q.s];
        q.e = a.off[q.s + 1];
    }
    if (q.end > a.rows) q.end = a.rows;
    return q;
}
__device__ __forceinline__ void mark_rows(const Args& a, int64_t row0, int nrows, const Marks& m, const Sequences& q) {
    for (int i = threadIdx.x; i < nrows / 16; i += NT) m.begin_bits[i] = 0;     // and the end bits behind
    __syncthreads();
    int64_t s = q.s, b = q.b, e = q.e;
    while (s < a.n && b < row0 + nrows) {
        if (e > b && b >= row0) {
            const int i = (int)(b - row0);
            m.begins[i] = (int32_t)s;
            atomicOr(&m.begin_bits[i >> 5], 1u << (i & 31));
        }
        if (e > b && e > row0 && e <= row0 + nrows) {
            const int i = (int)(e - 1 - row0);
            m.ends[i] = (int32_t)s;
            atomicOr(&m.end_bits[i >> 5], 1u << (i & 31));
        }
        s += NT;
        if (s < a.n) {
            b = a.off[s];
            e = a.off[s + 1];
        }
    }
    __syncthreads();
}
// Bits of the R rows from r0 on that lie in [first, end).
template <int R>
__device__ __forceinline__ uint32_t rows_within(int64_t r0, int64_t first, int64_t end) {
    const int64_t lo = first - r0, hi = end - r0;
    const uint32_t upto = hi <= 0 ? 0u : hi >= R ? (1u << R) - 1u : (1u << (int)hi) - 1u;
    const uint32_t before = lo <= 0 ? 0u : lo >= R ? (1u << R) - 1u : (1u << (int)lo) - 1u;
    return upto & ~before;
}

// ---- the state before a lane's rows -----------------------------------------------------------------
template <int VEC>
struct ScanLds {
    float a[W][64 * VEC], b[W][64 * VEC];
};

// The first `count` (at most N) words of a column, all asked for at once; unset ones, if the guard
// ever ran out, are NaN.
template <int N>
__device__ __forceinline__ void await(const uint64_t* p, int64_t stride, int count, uint64_t (&w)[N], bool& gave_up) {
    for (uint32_t looks = 0;; ++looks) {
        bool set = true;
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = i < count ? peek(p + i * stride) : 0;
#pragma unroll
        for (int i = 0; i < N; ++i) set = set && w[i] != kUnset;
        if (set) return;
        if (looks == kLooks) {
            gave_up = true;
            return;
        }
        __builtin_amdgcn_s_sleep(1);
    }
}

__device__ __forceinline__ uint64_t await_one(const uint64_t* p, bool& gave_up) {
    uint64_t w[1];
    await<1>(p, 0, 1, w, gave_up);
    return w[0];
}

// The state before a tile, for one channel a thread, given the tile's own step.  a.group (8) tiles form
// a group, whose last one publishes the group's step; as many groups form a row, and the state after
// those is passed on one by one.  (Groups of 16 that pass the state on themselves: 1000003 x 32 bf16
// 95 us, now 71; 200000 x 17 f32 with the gradient 101, now 80.  Rows of 16 groups of 16: 77 and 85.)
__device__ __forceinline__ Step thread_steps(const uint64_t* p, int64_t stride, int count, bool& gave_up) {
    Step s{1.0f, 0.0f};
    for (int j = 0; j < count; j += 4) {
        uint64_t w[4];
        await<4>(p + j * stride, stride, count - j, w, gave_up);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (j + i < count) s = after(s, Step{word_a(w[i]), word_b(w[i])});
    }
    return s;
}
__device__ __forceinline__ float carry_of_thread(const Args& a, int64_t tile, int64_t c, const Step& all,
                                                 bool& gave_up) {
    const int64_t g = tile / a.group, h = g / a.group;
    const int in_group = (int)(tile % a.group), in_groups = (int)(g % a.group);
    const bool last = in_group == a.group - 1, more = tile + 1 < a.ntiles;
    if (!last && more) publish(a.agg + tile * a.dp + c, word(all.a, all.b));
    const Step tiles = thread_steps(a.agg + g * a.group * a.dp + c, a.dp, in_group, gave_up);
    if (last && more) {
        const Step group = after(tiles, all);
        publish(a.inc + g * a.dp + c, word(group.a, group.b));
    }
    const Step groups = thread_steps(a.inc + h * a.group * a.dp + c, a.dp, in_groups, gave_up);
    const float row = h > 0 ? word_a(await_one(a.far + (h - 1) * a.dp + c, gave_up)) : 0.0f;
    const float carry = apply(tiles, apply(groups, row));
    if (last && in_groups == a.group - 1 && more) publish(a.far + h * a.dp + c, word(apply(all, carry), 0.0f));
    return carry;
}

// The same for one channel a wave, where there are few: a lane for each tile before in the group, then
// a lane for each group before; groups and rows are of 64.
__device__ __forceinline__ Step wave_steps(const uint64_t* p, int64_t stride, int count, bool& gave_up) {
    const int lane = threadIdx.x & 63;
    Step s{1.0f, 0.0f};
    if (lane < count) {
        const uint64_t w = await_one(p + lane * stride, gave_up);
        s = Step{word_a(w), word_b(w)};
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const Step q{__shfl_down(s.a, d), __shfl_down(s.b, d)};
        if ((lane & (2 * d - 1)) == 0) s = after(s, q);
    }
    return Step{__shfl(s.a, 0), __shfl(s.b, 0)};
}
__device__ __forceinline__ float carry_of_wave(const Args& a, int64_t tile, int64_t c, const Step& all,
                                               bool& gave_up) {
    const int64_t g = tile / 64, h = g / 64;
    const int in_group = (int)(tile % 64), in_groups = (int)(g % 64);
    const bool first = (threadIdx.x & 63) == 0, last = in_group == 63, more = tile + 1 < a.ntiles;
    if (first && !last && more) publish(a.agg + tile * a.dp + c, word(all.a, all.b));
    const Step tiles = wave_steps(a.agg + g * 64 * a.dp + c, a.dp, in_group, gave_up);
    const Step group = after(tiles, all);
    if (first && last && more) publish(a.inc + g * a.dp + c, word(group.a, group.b));
    const Step groups = wave_steps(a.inc + h * 64 * a.dp + c, a.dp, in_groups, gave_up);
    const float row = h > 0 ? word_a(await_one(a.far + (h - 1) * a.dp + c, gave_up)) : 0.0f;
    const float carry = apply(tiles, apply(groups, row));
    if (first && last && in_groups == 63 && more) publish(a.far + h * a.dp + c, word(apply(all, carry), 0.0f));
    return carry;
}

// From the steps of every lane's rows to the state before them: lanes of a wave by shuffles, the
// waves and the tiles before by a thread (or a wave) for each channel.
template <int VEC>
__device__ __forceinline__ void chain(const Args& a, const Place& at, const Step (&own)[VEC], ScanLds<VEC>& l,
                                      float (&h)[VEC]) {
    bool gave_up = false;
    const int cl = 1 << a.cl_bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int cols = cl * VEC, mine = (lane & (cl - 1)) * VEC;
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
            l.a[wave][mine + v] = s[v].a;
            l.b[wave][mine + v] = s[v].b;
        }
    }
    if (cl < 64) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            s[v] = Step{__shfl_up(s[v].a, cl), __shfl_up(s[v].b, cl)};
            if (lane < cl) s[v] = Step{1.0f, 0.0f};
        }
    }
    __syncthreads();
    const bool waves = cols <= W;
    const int col = waves ? wave : (int)threadIdx.x;
    if (col < cols) {
        Step all{1.0f, 0.0f};
#pragma unroll 2
        for (int w = 0; w < W; ++w) all = after(all, Step{l.a[w][col], l.b[w][col]});
        float carry = 0.0f;
        if (a.tickets) {
            const int64_t c = (int64_t)at.block * cols + col;
            carry = waves ? carry_of_wave(a, at.tile, c, all, gave_up) : carry_of_thread(a, at.tile, c, all, gave_up);
        }
#pragma unroll 2
        for (int w = 0; w < W; ++w) {
            const float next = apply(Step{l.a[w][col], l.b[w][col]}, carry);
            if (!waves || lane == 0) l.b[w][col] = carry;
            carry = next;
        }
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        h[v] = l.b[wave][mine + v];
        if (cl < 64) h[v] = apply(s[v], h[v]);
    }
    if (gave_up) tell_gave_up();             // here, where registers are free
}

// A lane's entries of a row: the row's address is the same in all lanes, and each lane's offset from
// it the same in all rows (one register; check_tile keeps it under 2^31).
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> load(const char* row, uint32_t offset) {
    Raw<T, VEC> r;
    r.load(row + offset);
    return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store(char* row, uint32_t offset, const float (&f)[VEC]) {
    struct alignas(sizeof(typename T::E) * VEC) Out {
        typename T::E e[VEC];
    } o;
#pragma unroll
    for (int v = 0; v < VEC; ++v) o.e[v] = (typename T::E)f[v];
    *(Out*)(row + offset) = o;
}
// The gates of VEC channels: their own, or one that they share.
template <typename L, int VEC, bool OWN>
struct Gates {
    Raw<L, OWN ? VEC : 1> r;
    static __device__ __forceinline__ uint32_t column(const Args& a, int c) {
        return (uint32_t)((OWN ? c : c / a.share) * (int)sizeof(typename L::E));
    }
    __device__ __forceinline__ void load_row(const char* row, uint32_t offset) { r = load<L, OWN ? VEC : 1>(row, offset); }
    __device__ __forceinline__ float operator[](int v) const { return r[OWN ? v : 0]; }
};

// ---- launch shapes ---------------------------------------------------------------------------------
struct Shape {
    int vec, cl_bits, ncb, r, group, dl_width, dl_parts;
    int64_t ntiles, dp;
    int64_t words() const { return ntiles > 1 ? (ntiles + groups() + ceil_div(groups(), group)) * dp : 0; }
    int64_t groups() const { return ceil_div(ntiles, group); }
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
    // or makes a tile's marks outgrow 34 KB of LDS
    s.r = grad ? 8 : 16;                              // four operands a row, not two
    if (ceil_div(rows, tg * s.r) * s.ncb < 256 || tg * s.r > 4096) s.r = 4;
    s.ntiles = ceil_div(rows, (int64_t)tg * s.r);
    s.group = (vec << s.cl_bits) > W ? 8 : 64;       // a thread's words in turn, a wave's at once
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
inline int wide_vec(int32_t dtype) { return 4 / elem_size(dtype); }

// 4 bytes of x a lane (and a row) where every operand's rows are aligned for it and no such piece
// has two gates; else an entry a lane.  Wider pieces would leave fewer rows to a lane's registers,
// and so make more tiles of the same rows.
inline int vec_of(int32_t dtype, int32_t gate_dtype, int32_t h_dtype, int d, int share,
                  std::initializer_list<const void*> x, std::initializer_list<int64_t> ld, const void* h, int64_t ld_h,
                  const void* l, int64_t ld_l, const void* dl, int64_t ld_dl) {
    const int v = wide_vec(dtype), es = elem_size(dtype), gs = elem_size(gate_dtype), hs = elem_size(h_dtype);
    if (v == 1 || d % v || (share > 1 && share % v)) return 1;
    for (const void* p : x)
        if ((uintptr_t)p % 4) return 1;
    for (int64_t s : ld)
        if (s * es % 4) return 1;
    if ((uintptr_t)h % (v * hs) || ld_h * hs % (v * hs)) return 1;
    if (share == 1 && ((uintptr_t)l % (v * gs) || ld_l * gs % (v * gs) || (uintptr_t)dl % (v * gs) || ld_dl * gs % (v * gs)))
        return 1;
    return v;
}

// f(type of x, type of h, type of the gates, channels a lane, whether each has a gate of its own)
template <typename X, typename H, typename L, typename F>
void with_vec(int vec, bool own, F f) {
    if constexpr (sizeof(typename X::E) == 2) {
        using two = std::integral_constant<int, 2>;
        if (vec == 2 && own) return f(X(), H(), L(), two(), std::true_type());
        if (vec == 2) return f(X(), H(), L(), two(), std::false_type());
    }
    f(X(), H(), L(), std::integral_constant<int, 1>(), std::false_type());      // its gate by its index
}
template <typename X, typename F>
void with_h(int32_t h_dtype, int32_t gate_dtype, int vec, bool own, F f) {
    if (h_dtype == DDM_F32)
        return gate_dtype == DDM_F32 ? with_vec<X, f32_t, f32_t>(vec, own, f) : with_vec<X, f32_t, X>(vec, own, f);
    return gate_dtype == DDM_F32 ? with_vec<X, X, f32_t>(vec, own, f) : with_vec<X, X, X>(vec, own, f);
}
template <typename F>
void with_types(int32_t dtype, int32_t h_dtype, int32_t gate_dtype, int vec, bool own, F f) {
    if (dtype == DDM_F32) return with_vec<f32_t, f32_t, f32_t>(vec, own, f);
    if (dtype == DDM_BF16) return with_h<bf16_t>(h_dtype, gate_dtype, vec, own, f);
    return with_h<f16_t>(h_dtype, gate_dtype, vec, own, f);
}

inline int check(const char* who, int32_t dtype, int32_t gate_dtype, int64_t rows, int64_t d, int64_t gates,
                 int64_t ld_x, int64_t ld_l, int64_t n, int32_t scale, int32_t flags) {
    if ((dtype != DDM_F32 && dtype != DDM_BF16 && dtype != DDM_F16) || (gate_dtype != dtype && gate_dtype != DDM_F32)) {
        set_error("%s: types %d and %d (gates of the inputs' type, or float32)", who, (int)dtype, (int)gate_dtype);
    } else if (rows < 0 || d < 1 || d > 1 << 20 || gates < 1 || d % gates || ld_x < d || (ld_l < gates && ld_l != 0) ||
               rows > (int64_t)1 << 40 || n < 0 || n > INT32_MAX) {
        set_error("%s: invalid argument (rows %lld, channels %lld, gates %lld that divide them, strides %lld and %lld)",
                  who, (long long)rows, (long long)d, (long long)gates, (long long)ld_x, (long long)ld_l);
    } else if (scale != DDM_GATED_NONE && scale != DDM_GATED_EWMA && scale != DDM_GATED_UNIT) {
        set_error("%s: unknown scale %d", who, (int)scale);
    } else if (flags & ~(DDM_GATED_FILL | DDM_GATED_H_F32)) {
        set_error("%s: unknown flags %d", who, (int)flags);
    } else {
        return 0;
    }
    return DDM_E_ARG;
}

// 0, or DDM_E_ARG where the grid has no room for the tiles, or a tile's rows lie too far apart for 32 bits.
inline int check_tile(const char* who, const Shape& s, std::initializer_list<int64_t> ld_bytes) {
    if (check_grid(who, s.ntiles * s.ncb + kQueues * kDies, NT)) {
        set_error("%s: %lld tiles of %d channel blocks (under 2^32 work-items a launch)", who, (long long)s.ntiles, s.ncb);
        return DDM_E_ARG;
    }
    const int64_t rows = (int64_t)(NT >> s.cl_bits) * s.r;
    for (int64_t ld : ld_bytes)
        if (ld > (((int64_t)1 << 31) - (4 << 20)) / rows) {
            set_error("%s: a row stride of %lld bytes (at most 2^31 / %lld)", who, (long long)ld, (long long)rows);
            return DDM_E_ARG;
        }
    return 0;
}

inline int64_t grid_of(const Args& a, const Shape& s) {
    return a.tickets ? queue_grid(s.ntiles * (s.ncb / a.queues), a.queues) : s.ntiles * s.ncb;
}

inline int64_t scratch_bytes(const Shape& s, int64_t rows, int d) {
    const int64_t parts = s.dl_parts ? rows * (d / (s.vec * s.dl_width)) : 0;
    return (s.words() ? kTicketBytes + 8 * s.words() : 0) + 4 * parts;
}

// The chain's buffers and the copy of the states, with their launch where either is needed (gated.hip).
int begin(Args& a, const Shape& s, void* scratch, const float* from, float* to, int64_t nstate, hipStream_t st);

}  // namespace gated
}  // namespace ddm
