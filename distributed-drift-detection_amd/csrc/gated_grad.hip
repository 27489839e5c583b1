// The recurrence's gradient (the method: gated.h).
#include "gated.h"

namespace ddm {
namespace gated {

// Rows in the opposite order: position p of the recurrence is row ntiles * tr - 1 - p, and a lane's
// rows run from its last one back; bits of rows count from the first, as in the forward.  Four operands
// a row leave room for 8 rows, and gates are computed again rather than kept, so three workgroups share
// a CU.  65536 x 2048 bf16, one sequence: 406 us, 4.0 TB/s ("unit" in 37 sequences 418); 16384 x 2048 bf16 with 128
// gates: 99 us.  Float32 gates of their own beside 16-bit inputs spill 12 registers: 529 us where the bytes at
// a copy's rate take 438 (16-bit gates: 418 and 329).
// h is of the inputs' type, half a step of which is then in the gates' gradients, or float32 (two workgroups
// a CU, as many bytes again for a 16-bit h): the caller's choice.  16384 x 2048 bf16 with 128 gates, one
// sequence: scan 49 -> 56 us, gradient 101 -> 123.
template <typename X, typename H, typename L, int VEC, bool OWN, int R>
__global__ __launch_bounds__(NT, (std::is_same<X, H>::value ? 6 : 4)) void k_gated_grad(Args a) {
    extern __shared__ int32_t marks[];
    __shared__ ScanLds<VEC> lds;
    const Place at = take(a);
    if (at.tile >= a.ntiles) return;
    const int cl = 1 << a.cl_bits, tg = (NT >> a.cl_bits) - 1 - (threadIdx.x >> a.cl_bits);
    const int tr = (NT >> a.cl_bits) * R;
    const int c = (at.block * cl + (int)(threadIdx.x & (cl - 1))) * VEC;
    const int64_t row0 = (a.ntiles - 1 - at.tile) * tr, r0 = row0 + tg * R;
    const bool active = c < a.d;
    Sequences seq{};
    if (a.off) seq = find_sequences(a, row0);
    Raw<X, VEC> x[R], dh[R];
    Raw<H, VEC> hp[R];
    Gates<L, VEC, OWN> l[R];
    auto lane_of = [&](int64_t ld) { return tg * R * (uint32_t)ld + c * (uint32_t)sizeof(typename X::E); };
    const uint32_t lane_x = lane_of(a.ld_x), lane_dh = lane_of(a.ld_dh);
    const uint32_t lane_h = tg * R * (uint32_t)a.ld_h + c * (uint32_t)sizeof(typename H::E);
    const uint32_t column_l = Gates<L, VEC, OWN>::column(a, c), lane_l = tg * R * (uint32_t)a.ld_l + column_l;
    auto load_row = [&](int r) {
        const int64_t row = row0 + r;                 // of the first time group
        dh[r] = load<X, VEC>(a.dh + row * a.ld_dh, lane_dh);
        l[r].load_row(a.l + row * a.ld_l, lane_l);
        x[r] = load<X, VEC>(a.x + row * a.ld_x, lane_x);
        if (r0 + r > 0) hp[r] = load<H, VEC>(a.h + (row - 1) * a.ld_h, lane_h);
    };
    if (row0 + tr <= a.rows) {
        if (active)
#pragma unroll
            for (int r = 0; r < R; ++r) load_row(r);
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (active && r0 + r < a.rows) load_row(r);
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
    const bool plain = !__any(active && (begins || ends || inside != (1u << R) - 1u));
    auto given = [&](int r, int v) {
        const int64_t s = a.off ? m.ends[tg * R + r] : 0;
        return a.dstate ? a.dstate[s * a.d + c + v] : 0.0f;
    };

    Step own[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) own[v] = Step{1.0f, 0.0f};
#pragma unroll
    for (int r = R - 1; r >= 0; --r)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float g = bounded_gate_of<DDM_GATED_NONE>(l[r][v]).a, y = dh[r][v];
            if (plain) {
                own[v].a *= g;
                own[v].b = g * (own[v].b + y);
            } else {
                Step q{kCut, 0.0f};
                if (active && inside >> r & 1)
                    q = ends >> r & 1 ? Step{kCut, g * (y + given(r, v))} : Step{g, g * y};
                own[v] = after(own[v], q);
            }
        }
    float u[VEC];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        dh[r].forget();
        l[r].r.forget();
    }
    chain<VEC>(a, at, own, lds, u);
    auto put = [&](int r, const float (&dx)[VEC], const float (&dl)[VEC], bool here) {
        const int64_t row = r0 + r;
        if (here) store<X, VEC>(a.dx + (row0 + r) * a.ld_dx, lane_of(a.ld_dx), dx);
        if (OWN) {
            if (here) store<L, VEC>(a.dl + (row0 + r) * a.ld_dl, tg * R * (uint32_t)a.ld_dl + column_l, dl);
            return;
        }
        float sum = dl[0];
#pragma unroll
        for (int v = 1; v < VEC; ++v) sum += dl[v];
        for (int k = 1; k < a.dl_width; k <<= 1) sum += __shfl_xor(sum, k);
        if (here && (threadIdx.x & (a.dl_width - 1)) == 0) {
            if (a.dl_part)
                a.dl_part[row * (a.d / (VEC * a.dl_width)) + c / (VEC * a.dl_width)] = sum;
            else
                *(typename L::E*)(a.dl + row * a.ld_dl + column_l) = (typename L::E)sum;
        }
    };
    with_scale(a.scale, [&](auto scale) {
        if (plain) {
#pragma unroll
            for (int r = R - 1; r >= 0; --r) {
                float dx[VEC], dl[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const Gate q = bounded_gate_of<scale()>(l[r][v]);
                    const float grad = dh[r][v] + u[v];
                    dx[v] = grad * q.f;
                    dl[v] = grad * fmaf(slope_of<scale()>(q), x[r][v], q.a * hp[r][v]);
                    u[v] = q.a * grad;
                }
                put(r, dx, dl, active);
            }
            return;
        }
#pragma unroll
        for (int r = R - 1; r >= 0; --r) {
            const bool in = active && inside >> r & 1;
            float dx[VEC], dl[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                dx[v] = dl[v] = 0.0f;
                if (!in) {
                    u[v] = 0.0f;
                    continue;
                }
                const Gate q = bounded_gate_of<scale()>(l[r][v]);
                const float grad = dh[r][v] + (ends >> r & 1 ? given(r, v) : u[v]);
                float before = hp[r][v];
                u[v] = q.a * grad;
                if (begins >> r & 1) {
                    const int64_t s = a.off ? m.begins[tg * R + r] : 0;
                    before = a.state_in ? a.state_in[s * a.d + c + v] : 0.0f;
                    a.state_out[s * a.d + c + v] = u[v];
                }
                dx[v] = grad * q.f;
                dl[v] = grad * fmaf(slope_of<scale()>(q), x[r][v], q.a * before);
            }
            put(r, dx, dl, in || (a.fill && active && r0 + r < a.rows));
        }
    });
}

// Gates shared by more channels than a wave sums: the parts of each, in order.  An odd number of channels a gate
// leaves every channel a part: 8192 x 1001 bf16 with one gate 344 us, gradient and sums, x 1024 48; 65536 x 1023
// with 341 gates 404, 65536 x 1024 with 256 183.
template <typename L>
__global__ __launch_bounds__(256) void k_gated_sum(Args a, int64_t gates, int per) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / gates, g = i % gates;
    int64_t first = 0, end = a.rows;
    if (a.off) {
        first = a.off[0];
        end = a.off[a.n];
    }
    if (row >= a.rows || (!a.fill && (row < first || row >= end))) return;
    const float* p = a.dl_part + (row * gates + g) * per;
    float sum = 0.0f;
    for (int k = 0; k < per; ++k) sum += p[k];
    *(typename L::E*)(a.dl + row * a.ld_dl + g * sizeof(typename L::E)) = (typename L::E)sum;
}

}  // namespace gated

int use_guard_gated_grad(bool* gave_up) { return use_guard(nullptr, gave_up); }
}  // namespace ddm

using namespace ddm;
using namespace ddm::gated;

extern "C" int ddm_gated_scan_grad(const void* x, int32_t dtype, int64_t ld_x, const void* log_a, int32_t gate_dtype,
                                   int64_t ld_a, const void* h, int64_t ld_h, const void* d_h, int64_t ld_dh,
                                   int64_t rows, int64_t d, int64_t gates, const int64_t* offsets, int64_t n,
                                   int32_t scale, const float* state_in, const float* d_state_out, float* d_state_in,
                                   void* d_x, int64_t ld_dx, void* d_log_a, int64_t ld_da, int32_t flags, void* scratch,
                                   ddm_stream_t stream, ddm_event_t ev_begin, ddm_event_t ev_end) {
    if (int rc = check("ddm_gated_scan_grad", dtype, gate_dtype, rows, d, gates, ld_x, ld_a, n, scale, flags)) return rc;
    if ((rows && (!x || !log_a || !h || !d_h || !d_x || !d_log_a || ld_h < d || ld_dh < d || ld_dx < d || ld_da < gates)) ||
        (n && !d_state_in) || (!offsets && n != 1) || (d_state_out && d_state_out == d_state_in)) {
        set_error("ddm_gated_scan_grad: invalid argument (null pointer, stride, one sequence without offsets, or the "
                  "states in one buffer)");
        return DDM_E_ARG;
    }
    const int32_t h_dtype = flags & DDM_GATED_H_F32 ? DDM_F32 : dtype;
    const int share = (int)(d / gates), es = elem_size(dtype), gs = elem_size(gate_dtype), hs = elem_size(h_dtype);
    const int vec = vec_of(dtype, gate_dtype, h_dtype, (int)d, share, {x, d_h, d_x}, {ld_x, ld_dh, ld_dx}, h, ld_h, log_a,
                           ld_a, d_log_a, ld_da);
    const Shape s = shape_of(rows, (int)d, share, vec, true);
    if (int rc = check_tile("ddm_gated_scan_grad", s,
                            {ld_x * es, ld_a * gs, ld_h * hs, ld_dh * es, ld_dx * es, ld_da * gs}))
        return rc;
    const int64_t sums = s.dl_parts ? ceil_div(rows * gates, 256) : 0;
    if (int rc = check_grid("ddm_gated_scan_grad", sums, 256)) return rc;
    if (scratch_bytes(s, rows, (int)d) && !scratch) {
        set_error("ddm_gated_scan_grad: invalid argument (no scratch)");
        return DDM_E_ARG;
    }
    const hipStream_t st = as_hip(stream);
    return timed(ev_begin, ev_end, st, [&]() -> int {
        Args a{};
        a.x = (const char*)x;
        a.l = (const char*)log_a;
        a.h = (const char*)h;
        a.dh = (const char*)d_h;
        a.dx = (char*)d_x;
        a.dl = (char*)d_log_a;
        a.ld_x = ld_x * es;
        a.ld_l = ld_a * gs;
        a.ld_h = ld_h * hs;
        a.ld_dh = ld_dh * es;
        a.ld_dx = ld_dx * es;
        a.ld_dl = ld_da * gs;
        a.rows = rows;
        a.d = (int)d;
        a.share = share;
        a.scale = scale;
        a.fill = flags & DDM_GATED_FILL;
        a.off = offsets;
        a.n = n;
        a.state_in = state_in;
        a.dstate = d_state_out;
        a.state_out = d_state_in;
        if (int rc = begin(a, s, scratch, d_state_out, d_state_in, n * d, st)) return rc;
        if (rows == 0) return 0;
        const size_t lds = offsets ? Marks::bytes((NT >> s.cl_bits) * s.r) : 0;
        const dim3 grid((unsigned)grid_of(a, s));
        int rc = 0;
        with_types(dtype, h_dtype, gate_dtype, vec, share == 1, [&](auto xt, auto ht, auto lt, auto v, auto own) {
            using X = decltype(xt);
            using H = decltype(ht);
            using L = decltype(lt);
            if (s.r == 8)
                k_gated_grad<X, H, L, v(), own(), 8><<<grid, NT, lds, st>>>(a);
            else
                k_gated_grad<X, H, L, v(), own(), 4><<<grid, NT, lds, st>>>(a);
            rc = launch_status("ddm_gated_scan_grad");
            if (!rc && sums) k_gated_sum<L><<<dim3((unsigned)sums), 256, 0, st>>>(a, gates, s.dl_parts);
        });
        return rc ? rc : launch_status("ddm_gated_scan_grad");
    });
}
