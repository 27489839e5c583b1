// The recurrence's gradient (the method: gated.h).
#include "gated.h"

namespace ddm {
namespace gated {

// ---- gradient ----------------------------------------------------------------------------------------
// Rows in the opposite order: position p of the recurrence is row ntiles * tr - 1 - p.
template <typename X, typename L, int VEC, bool OWN, int R>
__global__ __launch_bounds__(NT) void k_gated_grad(Args a) {
    extern __shared__ int32_t marks[];
    __shared__ ScanLds<VEC> lds;
    const Place at = take(a);
    const int cl = 1 << a.cl_bits, tg = threadIdx.x >> a.cl_bits, tr = (NT >> a.cl_bits) * R;
    const int c = (at.block * cl + (int)(threadIdx.x & (cl - 1))) * VEC;
    const int64_t row0 = (a.ntiles - 1 - at.tile) * tr, top = row0 + tr - 1 - tg * R;    // the lane's last row
    const bool active = c < a.d;
    Raw<X, VEC> x[R], dh[R], hp[R];
    Gates<L, VEC, OWN> l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t row = top - r;
        if (active && row < a.rows) {
            x[r] = load<X, VEC>(a.x, a.ld_x, row, c);
            l[r].load_row(a, row, c);
            dh[r] = load<X, VEC>(a.dh, a.ld_dh, row, c);
            if (row > 0) hp[r] = load<X, VEC>(a.h, a.ld_h, row - 1, c);
        }
    }
    int32_t *begins = marks, *ends = marks + tr;
    int64_t first = 0, end = a.rows;
    if (a.off) {
        mark_rows(a, row0, tr, begins, ends);
        first = a.off[0];
        end = a.off[a.n];
        end = end < a.rows ? end : a.rows;
    }
    auto inside = [&](int64_t row) { return active && row >= first && row < end; };
    auto ends_at = [&](int64_t row) { return a.off ? ends[row - row0] : row == a.rows - 1 ? 0 : -1; };
    auto given = [&](int s, int v) { return a.dstate ? a.dstate[(int64_t)s * a.d + c + v] : 0.0f; };
    Step own[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) own[v] = Step{1.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t row = top - r;
        const bool in = inside(row);
        const int s = in ? ends_at(row) : -1;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            Step q{kCut, 0.0f};
            if (in) {
                const float g = gate(l[r][v]), y = (float)dh[r].e[v];
                q = s >= 0 ? Step{kCut, g * (y + given(s, v))} : Step{g, g * y};
            }
            own[v] = after(own[v], q);
        }
    }
    float u[VEC];
    chain<VEC>(a, at, own, lds, u);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t row = top - r;
        const bool in = inside(row), put = in || (a.fill && active && row < a.rows);
        const int s_end = in ? ends_at(row) : -1;
        const int s_begin = !in ? -1 : a.off ? begins[row - row0] : row == 0 ? 0 : -1;
        float dx[VEC], dl[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            dx[v] = dl[v] = 0.0f;
            if (in) {
                const float lv = l[r][v], g = gate(lv), f = input_factor(lv, a.scale);
                const float grad = (float)dh[r].e[v] + (s_end >= 0 ? given(s_end, v) : u[v]);
                const float before = s_begin < 0 ? (float)hp[r].e[v]
                                     : a.state_in ? a.state_in[(int64_t)s_begin * a.d + c + v] : 0.0f;
                dx[v] = grad * f;
                dl[v] = grad * fmaf(input_slope(g, f, a.scale), (float)x[r].e[v], g * before);
                u[v] = g * grad;
                if (s_begin >= 0) a.state_out[(int64_t)s_begin * a.d + c + v] = u[v];
            } else {
                u[v] = 0.0f;
            }
        }
        if (put) store<X, VEC>(a.dx, a.ld_dx, row, c, dx);
        if (OWN) {
            if (put) store<L, VEC>(a.dl, a.ld_dl, row, c, dl);
        } else {
            float sum = dl[0];
#pragma unroll
            for (int v = 1; v < VEC; ++v) sum += dl[v];
            for (int k = 1; k < a.dl_width; k <<= 1) sum += __shfl_xor(sum, k);
            if (put && (threadIdx.x & (a.dl_width - 1)) == 0) {
                if (a.dl_part) {
                    const int64_t parts = a.d / (VEC * a.dl_width);
                    a.dl_part[row * parts + c / (VEC * a.dl_width)] = sum;
                } else {
                    *(typename L::E*)(a.dl + row * a.ld_dl + (int64_t)(c / a.share) * sizeof(typename L::E)) =
                        (typename L::E)sum;
                }
            }
        }
    }
}

// Gates shared by more channels than a wave sums: the parts of each, in order.
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
}  // namespace ddm

using namespace ddm;
using namespace ddm::gated;

extern "C" int ddm_gated_scan_grad(const void* x, int32_t dtype, int64_t ld_x, const void* log_a, int32_t gate_dtype,
                                   int64_t ld_a, const void* h, int64_t ld_h, const void* d_h, int64_t ld_dh,
                                   int64_t rows, int64_t d, int64_t gates, const int64_t* offsets, int64_t n,
                                   int32_t scale, const float* state_in, const float* d_state_out, float* d_state_in,
                                   void* d_x, int64_t ld_dx, void* d_log_a, int64_t ld_da, int32_t fill, void* scratch,
                                   ddm_stream_t stream, ddm_event_t ev_begin, ddm_event_t ev_end) {
    if (int rc = check("ddm_gated_scan_grad", dtype, gate_dtype, rows, d, gates, ld_x, ld_a, n, scale)) return rc;
    if ((rows && (!x || !log_a || !h || !d_h || !d_x || !d_log_a || ld_h < d || ld_dh < d || ld_dx < d || ld_da < gates)) ||
        (n && !d_state_in) || (!offsets && n != 1) || (d_state_out && d_state_out == d_state_in)) {
        set_error("ddm_gated_scan_grad: invalid argument (null pointer, stride, one sequence without offsets, or the "
                  "states in one buffer)");
        return DDM_E_ARG;
    }
    const int share = (int)(d / gates), es = elem_size(dtype), gs = elem_size(gate_dtype);
    const int vec = vec_of(dtype, gate_dtype, (int)d, share, {x, h, d_h, d_x}, {ld_x, ld_h, ld_dh, ld_dx}, log_a, ld_a,
                           d_log_a, ld_da);
    const Shape s = shape_of(rows, (int)d, share, vec, true);
    if (int rc = check_grid("ddm_gated_scan_grad", s)) return rc;
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
        a.ld_h = ld_h * es;
        a.ld_dh = ld_dh * es;
        a.ld_dx = ld_dx * es;
        a.ld_dl = ld_da * gs;
        a.rows = rows;
        a.d = (int)d;
        a.share = share;
        a.scale = scale;
        a.fill = fill;
        a.off = offsets;
        a.n = n;
        a.state_in = state_in;
        a.dstate = d_state_out;
        a.state_out = d_state_in;
        if (int rc = begin(a, s, scratch, d_state_out, d_state_in, n * d, st)) return rc;
        if (rows == 0) return 0;
        const size_t lds = offsets ? (size_t)(NT >> s.cl_bits) * s.r * 8 : 0;
        return with_types(dtype, gate_dtype, [&](auto xt, auto lt) {
            using X = decltype(xt);
            using L = decltype(lt);
            with_vec(vec, share == 1, [&](auto v, auto own) {
                constexpr int V = v() ? 1 : 8 / (int)sizeof(typename X::E);
                const dim3 grid((unsigned)(s.ntiles * s.ncb));
                if (s.r == 8)
                    k_gated_grad<X, L, V, own(), 8><<<grid, NT, lds, st>>>(a);
                else
                    k_gated_grad<X, L, V, own(), 2><<<grid, NT, lds, st>>>(a);
            });
            if (int rc = launch_status("ddm_gated_scan_grad")) return rc;
            if (s.dl_parts) {
                const int64_t blocks = ceil_div(rows * gates, 256);
                if (blocks > INT32_MAX) {
                    set_error("ddm_gated_scan_grad: %lld gate gradients", (long long)(rows * gates));
                    return DDM_E_ARG;
                }
                k_gated_sum<L><<<dim3((unsigned)blocks), 256, 0, st>>>(a, gates, s.dl_parts);
            }
            return launch_status("ddm_gated_scan_grad");
        });
    });
}
