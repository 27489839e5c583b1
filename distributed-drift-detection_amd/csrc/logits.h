// Rows of logits in registers: types, guarded wide loads, the running softmax of a lane and
// the merges of its parts (token_scores.hip, distill.hip).
#pragma once
#include <float.h>

#include <type_traits>

#include "common.h"

namespace ddm {
namespace logits {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// exp2 of anything at or below this is 0 in float32; products e * d take d clamped here, so
// that a masked entry (d = -inf, e = 0) adds 0 and not 0 * inf.  (The instruction gives 0 under 2^-126: a
// probability that float32 holds with fewer bits counts as none.)
constexpr float kDead = -200.0f;

struct f32_t {
    static constexpr int kCode = DDM_F32, kSize = 4, kVec = 4;
    static constexpr uint32_t kNegInf = 0xff800000u;     // one 32-bit word of -inf entries
    static __device__ __forceinline__ float one(const char* p) { return *(const float*)p; }
    static __device__ __forceinline__ uint32_t bits(const char* p) { return *(const uint32_t*)p; }
    static __device__ __forceinline__ void store(char* p, float v) { *(float*)p = v; }
};
struct bf16_t {
    static constexpr int kCode = DDM_BF16, kSize = 2, kVec = 8;
    static constexpr uint32_t kNegInf = 0xff80ff80u;
    static __device__ __forceinline__ float one(const char* p) {
        return __uint_as_float((uint32_t)*(const uint16_t*)p << 16);
    }
    static __device__ __forceinline__ uint32_t bits(const char* p) { return *(const uint16_t*)p; }
    static __device__ __forceinline__ void store(char* p, float v) { *(__bf16*)p = (__bf16)v; }
};
struct f16_t {
    static constexpr int kCode = DDM_F16, kSize = 2, kVec = 8;
    static constexpr uint32_t kNegInf = 0xfc00fc00u;
    static __device__ __forceinline__ float one(const char* p) { return (float)*(const _Float16*)p; }
    static __device__ __forceinline__ uint32_t bits(const char* p) { return *(const uint16_t*)p; }
    static __device__ __forceinline__ void store(char* p, float v) { *(_Float16*)p = (_Float16)v; }
};

// 16 bytes of entries as float32.
__device__ __forceinline__ void unpack(const uint4& r, float (&f)[4], f32_t) {
    f[0] = __uint_as_float(r.x);
    f[1] = __uint_as_float(r.y);
    f[2] = __uint_as_float(r.z);
    f[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void unpack(const uint4& r, float (&f)[8], bf16_t) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(const uint4& r, float (&f)[8], f16_t) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h2 h;
        __builtin_memcpy(&h, &w[i], 4);
        f[2 * i] = (float)h.x;
        f[2 * i + 1] = (float)h.y;
    }
}
// ... and back, rounded to nearest even once.
__device__ __forceinline__ uint4 pack(const float (&f)[4], f32_t) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <typename H>
__device__ __forceinline__ uint4 pack_half(const float (&f)[8]) {
    typedef H h2 __attribute__((ext_vector_type(2)));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2 h = {(H)f[2 * i], (H)f[2 * i + 1]};
        __builtin_memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], bf16_t) { return pack_half<__bf16>(f); }
__device__ __forceinline__ uint4 pack(const float (&f)[8], f16_t) { return pack_half<_Float16>(f); }

// A row as 16-byte aligned vectors: vector j holds the columns j*kVec - head + [0, kVec), of
// which those outside [0, v) are no entries.  Rows of an odd length start at any entry, so
// `head` differs from row to row; only vectors that lie wholly inside are loaded as one,
// the two at the ends entry by entry, and nothing outside the row is touched.
// How many vectors the longest row of a matrix takes: one more if rows need not start aligned.
inline int64_t vectors_of(const void* base, int64_t ld_bytes, int64_t v, int vec) {
    const bool aligned = ((uintptr_t)base & 15) == 0 && ld_bytes % 16 == 0;
    return ceil_div(v + (aligned ? 0 : vec - 1), vec);
}

template <typename T>
struct Row {
    const char* base;    // address of column 0
    int v;
    int head;            // entries between the aligned address below base and base
    __device__ __forceinline__ Row(const char* p, int64_t n) : base(p), v((int)n) {
        head = (int)(((uintptr_t)p & 15) / T::kSize);
    }
    __device__ __forceinline__ int col(int j) const { return j * T::kVec - head; }
    __device__ __forceinline__ int vector_of(int c) const { return (c + head) / T::kVec; }
    __device__ __forceinline__ bool whole(int j) const { return col(j) >= 0 && col(j) + T::kVec <= v; }
    __device__ __forceinline__ uint4 load_whole(int j) const { return *(const uint4*)(base + col(j) * T::kSize); }
    __device__ __forceinline__ float at(int c) const { return T::one(base + c * T::kSize); }
    __device__ __forceinline__ uint4 load(int j) const {
        if (whole(j)) return load_whole(j);
        uint32_t w[4] = {T::kNegInf, T::kNegInf, T::kNegInf, T::kNegInf};
        const int c0 = col(j);
        if (c0 < v) {
#pragma unroll
            for (int e = 0; e < T::kVec; ++e) {
                const int c = c0 + e;
                if (c >= 0 && c < v) {
                    const uint32_t b = T::bits(base + c * T::kSize);
                    if (T::kSize == 4)
                        w[e & 3] = b;
                    else
                        w[e >> 1] = (e & 1) ? (w[e >> 1] & 0xffffu) | (b << 16) : (w[e >> 1] & 0xffff0000u) | b;
                }
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // The vector's entries into another row (gradients), as one where that is aligned alike; but for
    // those with a bit in `without`.
    __device__ __forceinline__ void store(char* out, int j, const float (&f)[T::kVec], uint32_t without = 0) const {
        const int c0 = col(j);
        char* p = out + c0 * T::kSize;
        if (whole(j) && ((uintptr_t)p & 15) == 0 && without == 0) {
            *(uint4*)p = pack(f, T());
            return;
        }
#pragma unroll
        for (int e = 0; e < T::kVec; ++e)
            if (c0 + e >= 0 && c0 + e < v && !(without >> e & 1)) T::store(p + e * T::kSize, f[e]);
    }
};

// NV vectors a lane of the part of a row that starts at vector j0 (lane stride: NT vectors,
// so a wave's load covers 1 KB without a gap).  Parts without a row's end in them take the
// branch with plain loads, from one address and an offset a lane.
template <typename T, int NT, int NV>
__device__ __forceinline__ bool inside(const Row<T>& row, int j0) {
    return row.whole(j0) && row.whole(j0 + NT * NV - 1);
}
template <typename T, int NT, int NV>
__device__ __forceinline__ void load_part(const Row<T>& row, int j0, uint4 (&raw)[NV]) {
    if (inside<T, NT, NV>(row, j0)) {
        const char* p = row.base + row.col(j0) * T::kSize;
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = *(const uint4*)(p + i * NT * 16 + threadIdx.x * 16u);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = row.load(j0 + i * NT + (int)threadIdx.x);
    }
}
// The same part of another row (gradients): value(i, f) gives vector i, without(i) the bits of entries
// that are not to be written.
template <typename T, int NT, int NV, class Value, class Without>
__device__ __forceinline__ void store_part(const Row<T>& row, char* out, int j0, Value value, Without without) {
    const bool plain = inside<T, NT, NV>(row, j0) && (((uintptr_t)out ^ (uintptr_t)row.base) & 15) == 0;
    char* p = out + row.col(j0) * T::kSize;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[T::kVec];
        value(i, f);
        const uint32_t skip = without(i);
        if (plain && !__any(skip != 0))
            *(uint4*)(p + i * NT * 16 + threadIdx.x * 16u) = pack(f, T());
        else
            row.store(out, j0 + i * NT + (int)threadIdx.x, f, skip);
    }
}

// The same vector, but unknown to the compiler: what was computed from it before is not kept
// in registers for a later pass (eight floats a vector), which unpacks it again.
__device__ __forceinline__ uint4 again(uint4 r) {
    asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w));
    return r;
}

// A part's softmax: with d_i = (x_i - m) log2(e) / T over its entries, s = sum 2^d_i and
// u = sum 2^d_i d_i, for a reference m near its maximum.  m starts at the lowest finite value, so that -inf entries (d = -inf)
// add nothing and a part of them alone has s = 0; NaN and +inf make s NaN for good.
struct Part {
    float m, s, u;
};
__device__ __forceinline__ Part no_part() { return Part{-FLT_MAX, 0.0f, 0.0f}; }

// A lane's own running sums, an entry in four operations and the exponential.  d is one fused
// product, x log2(e) / T - scaled, with scaled = m log2(e) / T as float32 has it; what scaled lost in
// rounding (`lost`) is given back at the end (part_of), exactly.  m is a reference, not the maximum: it
// follows when an entry exceeds it by 8 binary orders (limit), which after a lane's first vector is
// seldom, and a sum of 2^8 is as exact as one of 1.
// scaled has to be known to a small part of one, so where it is over kWide (logits in the millions;
// rows masked by the type's lowest value and little else) d is (x - m) log2(e) / T instead, for the
// waves that have such lanes: their limit is -inf.
constexpr float kWide = 1048576.0f;
struct Lane {
    float m, scaled, limit, s, u;
};
__device__ __forceinline__ Lane no_lane() { return Lane{-FLT_MAX, -3e38f, -INFINITY, 0.0f, 0.0f}; }
__device__ __forceinline__ float lost(const Lane& l, float c) {
    return fabsf(l.scaled) > kWide ? 0.0f : -fmaf(l.m, c, -l.scaled);                       // scaled - m c
}
template <bool ENTROPY, int N>
__device__ __forceinline__ void add_vector(Lane& l, const float (&f)[N], float most, float c) {
    if (__any(most > l.limit)) {
        Lane to = l;
        if (most > l.limit) {
            to.m = fmaxf(l.m, most);
            to.scaled = fminf(fmaxf(to.m * c, -3e38f), 3e38f);
            // finite, so that +inf exceeds it at any temperature and leaves its NaN
            to.limit = fabsf(to.scaled) > kWide ? -INFINITY : fminf(to.m + 8.0f / c, FLT_MAX);
        }
        float d = l.scaled - to.scaled;
        if (__any(fabsf(l.scaled) > kWide || fabsf(to.scaled) > kWide))
            d = (l.m - to.m) * c + (lost(l, c) - lost(to, c));
        d = fmaxf(d, kDead);
        const float r = __builtin_amdgcn_exp2f(d);
        if (ENTROPY) to.u = r * fmaf(l.s, d, l.u);
        to.s = l.s * r;
        l = to;
        if (__any(fabsf(l.scaled) > kWide && most >= -FLT_MAX)) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float d = fabsf(l.scaled) > kWide ? (f[e] - l.m) * c : fmaf(f[e], c, -l.scaled);
                const float w = __builtin_amdgcn_exp2f(d);
                l.s += w;
                if (ENTROPY) l.u = fmaf(w, fmaxf(d, kDead), l.u);
            }
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float d = fmaf(f[e], c, -l.scaled);
        const float w = __builtin_amdgcn_exp2f(d);
        l.s += w;
        if (ENTROPY) l.u = fmaf(w, fmaxf(d, kDead), l.u);
    }
}
__device__ __forceinline__ Part part_of(const Lane& l, float c) {
    const float d = lost(l, c), r = __builtin_amdgcn_exp2f(d);
    return Part{l.m, l.s * r, fmaf(d, l.s, l.u) * r};
}
template <int N>
__device__ __forceinline__ float largest(const float (&f)[N]) {
    float m = f[0];
#pragma unroll
    for (int e = 1; e < N; ++e) m = fmaxf(m, f[e]);
    return m;
}

__device__ __forceinline__ void rebase(Part& a, float m, float c) {
    const float d = fmaxf((a.m - m) * c, kDead), r = __builtin_amdgcn_exp2f(d);
    a.u = r * fmaf(a.s, d, a.u);
    a.s *= r;
    a.m = m;
}
__device__ __forceinline__ Part merge(Part a, Part b, float c) {
    const float m = fmaxf(a.m, b.m);
    rebase(a, m, c);
    rebase(b, m, c);
    return Part{m, a.s + b.s, a.u + b.u};
}
__device__ __forceinline__ Part wave_merge(Part a, float c) {
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) {
        Part b;
        b.m = __shfl_xor(a.m, k);
        b.s = __shfl_xor(a.s, k);
        b.u = __shfl_xor(a.u, k);
        a = merge(a, b, c);
    }
    return a;
}

// ... and of a workgroup, in every lane.
template <int NT>
__device__ __forceinline__ Part block_merge(Part p, float c, Part* sh) {
    constexpr int W = NT / 64;
    p = wave_merge(p, c);
    if (W == 1) return p;
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = p;
    __syncthreads();
    const int lane = threadIdx.x & 63;
    return wave_merge(lane < W ? sh[lane] : no_part(), c);
}

// float32 as an unsigned integer of the same order (-0 as +0); -inf is kKeyNegInf.
constexpr uint32_t kKeyNegInf = 0x007fffffu;
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
// The next float32 below x (x finite).
__device__ __forceinline__ float below(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return __uint_as_float(b == 0u ? 0x80000001u : (b >> 31) ? b + 1u : b - 1u);
}

__device__ __forceinline__ int64_t target_at(const void* t, int wide, int64_t i) {
    return wide ? ((const int64_t*)t)[i] : (int64_t)((const int32_t*)t)[i];
}

constexpr int kMaxTop = 64;              // alternatives of a row: one a lane
constexpr int kMaxParts = 64;            // parts that a short list of rows is cut into, as well; the longest
                                         // float32 row that does not start aligned takes 65
constexpr int64_t kMaxColumns = 1 << 19;

struct Shape {
    int nt, nv, turns, parts;    // a workgroup's part: turns times nv vectors a lane
};
template <typename F>
int with_type(int32_t dtype, F f) {
    switch (dtype) {
        case DDM_F32: return f(f32_t());
        case DDM_BF16: return f(bf16_t());
        case DDM_F16: return f(f16_t());
    }
    return DDM_E_ARG;
}
#define DDM_SHAPE(NT_, NV_) \
    if (s.nt == NT_ && s.nv == NV_) return f(std::integral_constant<int, NT_>(), std::integral_constant<int, NV_>())
template <typename F>
void with_part_shape(const Shape& s, F f) {
    DDM_SHAPE(64, 1);
    DDM_SHAPE(64, 2);
    DDM_SHAPE(64, 4);
    DDM_SHAPE(64, 8);
    DDM_SHAPE(256, 1);
    DDM_SHAPE(256, 2);
    DDM_SHAPE(256, 4);
    DDM_SHAPE(256, 8);
}
#undef DDM_SHAPE

// The checks the entry points share; 0 or DDM_E_ARG with the reason.
inline int check_rows(const char* who, int32_t dtype, int64_t n, int64_t v, int64_t ld, int32_t target_bytes,
                      float temperature, int32_t top) {
    if (dtype != DDM_F32 && dtype != DDM_BF16 && dtype != DDM_F16) {
        set_error("%s: unknown type %d", who, (int)dtype);
    } else if (n < 0 || v < 1 || v > kMaxColumns || ld < v || n > INT32_MAX / kMaxParts - 64) {
        set_error("%s: invalid argument (rows %lld, columns %lld of 1..%lld, row stride %lld)", who, (long long)n,
                  (long long)v, (long long)kMaxColumns, (long long)ld);
    } else if (target_bytes != 4 && target_bytes != 8) {
        set_error("%s: targets of %d bytes (4 or 8)", who, (int)target_bytes);
    } else if (!(temperature >= FLT_MIN) || !(temperature < INFINITY)) {
        set_error("%s: temperature must be positive (a normal float32) and finite", who);
    } else if (top < 0 || top > kMaxTop) {
        set_error("%s: %d alternatives (0..%d)", who, (int)top, kMaxTop);
    } else {
        return 0;
    }
    return DDM_E_ARG;
}

}  // namespace logits
}  // namespace ddm
