// The recurrence forwards, and its single step (the method: gated.h).
#include "gated.h"

namespace ddm {
namespace gated {

// A tile's steps stay in registers, two float32 an entry; 16 rows a lane let two workgroups share a CU.
// 65536 x 2048 bf16, "unit", 37 sequences: 234 us, 3.4 TB/s; one sequence of them 210.  What is above
// the 165 us of the same kernel without the chain is tiles waiting for tiles, and 4 us the look for gates over 1.  (With the steps computed
// again after the wait, three workgroups fit a CU: "unit" 235 us, "none" no faster.)
template <typename X, typename H, typename L, int VEC, bool OWN, int R>
__global__ __launch_bounds__(NT, 4) void k_gated_scan(Args a) {
    extern __shared__ int32_t marks[];
    __shared__ ScanLds<VEC> lds;
    const Place at = take(a);
    if (at.tile >= a.ntiles) return;
    const int cl = 1 << a.cl_bits, tg = threadIdx.x >> a.cl_bits, tr = (NT >> a.cl_bits) * R;
    const int c = (at.block * cl + (int)(threadIdx.x & (cl - 1))) * VEC;
    const int64_t row0 = at.tile * tr, r0 = row0 + tg * R;
    const bool active = c < a.d;
    Sequences seq{};
    if (a.off) seq = find_sequences(a, row0);
    Raw<X, VEC> x[R];
    Gates<L, VEC, OWN> l[R];
    const uint32_t lane_x = tg * R * (uint32_t)a.ld_x + c * (uint32_t)sizeof(typename X::E);
    const uint32_t lane_h = tg * R * (uint32_t)a.ld_h + c * (uint32_t)sizeof(typename H::E);
    const uint32_t lane_l = tg * R * (uint32_t)a.ld_l + Gates<L, VEC, OWN>::column(a, c);
    const char *x0 = a.x + row0 * a.ld_x, *l0 = a.l + row0 * a.ld_l;
    char* h0 = a.out + row0 * a.ld_h;
    if (row0 + tr <= a.rows) {
        if (active)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                x[r] = load<X, VEC>(x0 + r * a.ld_x, lane_x);
                l[r].load_row(l0 + r * a.ld_l, lane_l);
            }
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (active && r0 + r < a.rows) {
                x[r] = load<X, VEC>(x0 + r * a.ld_x, lane_x);
                l[r].load_row(l0 + r * a.ld_l, lane_l);
            }
    }
    const Marks m(marks, tr);
    uint32_t begins, ends, inside;
    if (a.off) {
        mark_rows(a, row0, tr, m, seq);
        begins = Marks::lane<R>(m.begin_bits, tg * R);
        ends = Marks::lane<R>(m.end_bits, tg * R);
        inside = rows_within<R>(r0, seq.first, seq.end);
    } else {
        begins = r0 == 0;
        ends = a.rows - 1 >= r0 && a.rows - 1 < r0 + R ? 1u << (int)(a.rows - 1 - r0) : 0u;
        inside = rows_within<R>(r0, 0, a.rows);
    }
    begins &= inside;
    ends &= inside;
    constexpr int G = OWN ? VEC : 1;                 // gates a lane; a cut is one of all its channels
    float g[R][G], b[R][VEC];
    Step own[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) own[v] = Step{1.0f, 0.0f};
    uint64_t over = 0;                               // lanes with a gate over 1
    with_scale(a.scale, [&](auto scale) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float in[G];
#pragma unroll
            for (int k = 0; k < G; ++k) {
                const Gate q = gate_of<scale()>(l[r][k]);
                g[r][k] = q.a;
                over |= __ballot(q.a > 1.0f);
                in[k] = q.f;
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                b[r][v] = in[v % G] * x[r][v];
                own[v].a *= g[r][v % G];
                own[v].b = fmaf(g[r][v % G], own[v].b, b[r][v]);
            }
        }
    });
    const bool plain = !__any(active && (begins || ends || inside != (1u << R) - 1u)) && !(over & __ballot(active));
    if (!plain) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) own[v] = Step{1.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool in = active && inside >> r & 1, first = begins >> r & 1;
#pragma unroll
            for (int k = 0; k < G; ++k)
                if (g[r][k] > 1.0f) g[r][k] = __builtin_nanf("");
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                if (in && first) {                   // without a state as well: a NaN gate's 0 is NaN
                    const int64_t s = a.off ? m.begins[tg * R + r] : 0;
                    b[r][v] = fmaf(g[r][v % G], a.state_in ? a.state_in[s * a.d + c + v] : 0.0f, b[r][v]);
                }
                if (!in) b[r][v] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < G; ++k)
                if (!in || first) g[r][k] = kCut;
#pragma unroll
            for (int v = 0; v < VEC; ++v) own[v] = after(own[v], Step{g[r][v % G], b[r][v]});
        }
    }
    float h[VEC];
    chain<VEC>(a, at, own, lds, h);
    if (plain) {
        if (!active) return;
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = fmaf(g[r][v % G], h[v], b[r][v]);
            store<H, VEC>(h0 + r * a.ld_h, lane_h, h);
        }
        return;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = apply(Step{g[r][v % G], b[r][v]}, h[v]);
        if (active && (inside >> r & 1 || (a.fill && r0 + r < a.rows))) store<H, VEC>(h0 + r * a.ld_h, lane_h, h);
        if (active && ends >> r & 1) {
            const int64_t s = a.off ? m.ends[tg * R + r] : 0;
#pragma unroll
            for (int v = 0; v < VEC; ++v) a.state_out[s * a.d + c + v] = h[v];
        }
    }
}

// One row a sequence: elementwise, the state's row beside it.  256 x 2048 bf16: 3.6 us, a launch's time.
template <typename X, typename L, int VEC, bool OWN>
__global__ __launch_bounds__(256) void k_gated_step(Args a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int per = a.d / VEC;
    const int64_t row = i / per;
    const int c = (int)(i % per) * VEC;
    if (row >= a.rows) return;
    const Raw<X, VEC> x = load<X, VEC>(a.x + row * a.ld_x, c * (uint32_t)sizeof(typename X::E));
    Gates<L, VEC, OWN> l;
    l.load_row(a.l + row * a.ld_l, Gates<L, VEC, OWN>::column(a, c));
    float h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = a.state_in ? a.state_in[row * a.d + c + v] : 0.0f;
    with_scale(a.scale, [&](auto scale) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Gate q = bounded_gate_of<scale()>(l[v]);
            h[v] = fmaf(q.a, h[v], q.f * x[v]);
        }
    });
#pragma unroll
    for (int v = 0; v < VEC; ++v) a.state_out[row * a.d + c + v] = h[v];
    store<X, VEC>(a.out + row * a.ld_h, c * (uint32_t)sizeof(typename X::E), h);
}

// The chain's buffers, the copy of the states, and where both are needed their launch.
int begin(Args& a, const Shape& s, void* scratch, const float* from, float* to, int64_t nstate, hipStream_t st) {
    char* w = (char*)scratch;
    const int64_t words = s.words();
    if (words) {
        a.tickets = (uint32_t*)w;
        a.queues = s.ncb % 8 == 0 ? 8 : s.ncb % 4 == 0 ? 4 : s.ncb % 2 == 0 ? 2 : 1;
        a.agg = (uint64_t*)(w + kTicketBytes);
        a.inc = a.agg + s.ntiles * s.dp;
        a.far = a.inc + s.groups() * s.dp;
        w += kTicketBytes + 8 * words;
    }
    if (s.dl_parts) a.dl_part = (float*)w;
    a.cl_bits = s.cl_bits;
    a.ncb = s.ncb;
    a.group = s.group;
    a.ntiles = s.ntiles;
    a.dp = s.dp;
    a.dl_width = s.dl_width;
    if (!words && !a.off && s.ntiles) return 0;        // one tile, one sequence that has rows
    return reset_words(a.tickets, a.agg, words, from, to, nstate, st, "ddm_gated_scan");
}

}  // namespace gated

int use_guard_gated(bool* gave_up) { return use_guard(nullptr, gave_up); }
}  // namespace ddm

using namespace ddm;
using namespace ddm::gated;

extern "C" int64_t ddm_gated_scan_scratch_bytes(int64_t rows, int64_t d, int64_t gates, int32_t dtype, int32_t grad) {
    if (rows <= 0 || d < 1 || d > 1 << 20 || gates < 1 || d % gates || dtype < 0 || dtype > DDM_F16) return 0;
    // whichever way the operands are aligned
    int64_t most = 0;
    for (int vec : {1, wide_vec(dtype)})
        if (d % vec == 0 && (gates == d || d / gates % vec == 0)) {
            const int64_t b = scratch_bytes(shape_of(rows, (int)d, (int)(d / gates), vec, grad != 0), rows, (int)d);
            most = b > most ? b : most;
        }
    return most;
}

extern "C" int ddm_gated_scan(const void* x, int32_t dtype, int64_t ld_x, const void* log_a, int32_t gate_dtype,
                              int64_t ld_a, int64_t rows, int64_t d, int64_t gates, const int64_t* offsets, int64_t n,
                              int32_t scale, const float* state_in, float* state_out, void* out, int64_t ld_out,
                              int32_t flags, void* scratch, ddm_stream_t stream, ddm_event_t ev_begin, ddm_event_t ev_end) {
    if (int rc = check("ddm_gated_scan", dtype, gate_dtype, rows, d, gates, ld_x, ld_a, n, scale, flags)) return rc;
    if ((rows && (!x || !log_a || !out || ld_out < d)) || (n && !state_out) || (!offsets && n != 1) ||
        (state_in && state_in == state_out)) {
        set_error("ddm_gated_scan: invalid argument (null pointer, output stride, one sequence without offsets, or the "
                  "states in one buffer)");
        return DDM_E_ARG;
    }
    const int32_t h_dtype = flags & DDM_GATED_H_F32 ? DDM_F32 : dtype;
    const int share = (int)(d / gates), es = elem_size(dtype), gs = elem_size(gate_dtype), hs = elem_size(h_dtype);
    const int vec = vec_of(dtype, gate_dtype, h_dtype, (int)d, share, {x}, {ld_x}, out, ld_out, log_a, ld_a, nullptr, 0);
    const Shape s = shape_of(rows, (int)d, share, vec, false);
    if (int rc = check_tile("ddm_gated_scan", s, {ld_x * es, ld_a * gs, ld_out * hs})) return rc;
    if (scratch_bytes(s, rows, (int)d) && !scratch) {
        set_error("ddm_gated_scan: invalid argument (no scratch)");
        return DDM_E_ARG;
    }
    const hipStream_t st = as_hip(stream);
    return timed(ev_begin, ev_end, st, [&]() -> int {
        Args a{};
        a.x = (const char*)x;
        a.l = (const char*)log_a;
        a.out = (char*)out;
        a.ld_x = ld_x * es;
        a.ld_l = ld_a * gs;
        a.ld_h = ld_out * hs;
        a.rows = rows;
        a.d = (int)d;
        a.share = share;
        a.scale = scale;
        a.fill = flags & DDM_GATED_FILL;
        a.off = offsets;
        a.n = n;
        a.state_in = state_in;
        a.state_out = state_out;
        if (int rc = begin(a, s, scratch, state_in, state_out, n * d, st)) return rc;
        if (rows == 0) return 0;
        const size_t lds = offsets ? Marks::bytes((NT >> s.cl_bits) * s.r) : 0;
        const dim3 grid((unsigned)grid_of(a, s));
        with_types(dtype, h_dtype, gate_dtype, vec, share == 1, [&](auto xt, auto ht, auto lt, auto v, auto own) {
            using X = decltype(xt);
            using H = decltype(ht);
            using L = decltype(lt);
            if (s.r == 16)
                k_gated_scan<X, H, L, v(), own(), 16><<<grid, NT, lds, st>>>(a);
            else
                k_gated_scan<X, H, L, v(), own(), 4><<<grid, NT, lds, st>>>(a);
        });
        return launch_status("ddm_gated_scan");
    });
}

extern "C" int ddm_gated_step(const void* x, int32_t dtype, int64_t ld_x, const void* log_a, int32_t gate_dtype,
                              int64_t ld_a, int64_t rows, int64_t d, int64_t gates, int32_t scale, const float* state_in,
                              float* state_out, void* out, int64_t ld_out, ddm_stream_t stream, ddm_event_t ev_begin,
                              ddm_event_t ev_end) {
    if (int rc = check("ddm_gated_step", dtype, gate_dtype, rows, d, gates, ld_x, ld_a, rows, scale, 0)) return rc;
    if (rows == 0) return timed_nothing(ev_begin, ev_end, stream);
    if (!x || !log_a || !state_out || !out || ld_out < d) {
        set_error("ddm_gated_step: invalid argument (null pointer or output stride)");
        return DDM_E_ARG;
    }
    const int share = (int)(d / gates), es = elem_size(dtype), gs = elem_size(gate_dtype);
    auto in_state_out = [&](const void* p, int64_t bytes) {      // a row of it is read after another is written
        return (uintptr_t)p < (uintptr_t)(state_out + rows * d) && (uintptr_t)state_out < (uintptr_t)p + bytes;
    };
    if (in_state_out(x, ((rows - 1) * ld_x + d) * es) || in_state_out(log_a, ((rows - 1) * ld_a + gates) * gs)) {
        set_error("ddm_gated_step: the state after overlaps the inputs");
        return DDM_E_ARG;
    }
    const int vec = vec_of(dtype, gate_dtype, dtype, (int)d, share, {x}, {ld_x}, out, ld_out, log_a, ld_a, nullptr, 0);
    const int64_t blocks = ceil_div(rows * (d / vec), 256);
    if (int rc = check_grid("ddm_gated_step", blocks, 256)) return rc;
    const hipStream_t st = as_hip(stream);
    return timed(ev_begin, ev_end, st, [&] {
        Args a{};
        a.x = (const char*)x;
        a.l = (const char*)log_a;
        a.out = (char*)out;
        a.ld_x = ld_x * es;
        a.ld_l = ld_a * gs;
        a.ld_h = ld_out * es;
        a.rows = rows;
        a.d = (int)d;
        a.share = share;
        a.scale = scale;
        a.state_in = state_in;
        a.state_out = state_out;
        with_types(dtype, dtype, gate_dtype, vec, share == 1, [&](auto xt, auto, auto lt, auto v, auto own) {
            k_gated_step<decltype(xt), decltype(lt), v(), own()><<<dim3((unsigned)blocks), 256, 0, st>>>(a);
        });
        return launch_status("ddm_gated_step");
    });
}
