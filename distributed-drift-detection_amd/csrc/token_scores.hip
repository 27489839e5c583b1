// What a language model answered, for the drift scans: log probability, entropy, rank, error
// flag and the top alternatives of every row of logits, in one pass over them; and the
// gradient of weighted log probabilities, entropies and alternatives.
//
// With d_i = (x_i - m) / T, m near the row's maximum, S = sum e^d_i, U = sum e^d_i d_i:
//   log p_i = d_i - log S,   H = log S - U / S,   rank = #{x_i > x_t or x_i = x_t, i < t}.
// The pass is bound by reading the logits; what it computes per entry (12 vector instructions with
// the alternatives, one of them an exponential at a quarter of the rate) takes as long as that
// for 16-bit logits: 8192 x 131072 are 2.05e8 instructions of a wave, 4 cycles each on 1024 units at 2.4 GHz 335
// us, and 12 cycles more for each of 1.7e7 exponentials 80.  A row is cut into parts (shape_of), one a workgroup, so that several workgroups
// share a CU and one's sums run behind another's loads; few rows are cut finer, until there are
// enough workgroups for the chip.  Parts meet in a second small launch.  No atomic decides an
// order: every sum is a fixed tree, and the alternatives are ordered by (value, index).
// Measured: 8192 x 131072 bf16 with 32 alternatives 417 us, 5.2 TB/s; 4096 x 65536 bf16 without 142 us; 1000 x 50021 float32 with 5 50 us, 4.0 TB/s; one row of
// 131072 bf16 with 20 in 8 + 6.5 us, latencies of the two launches.  (A copy of 2 GB runs at
// 4.9 TB/s, reads and writes together.)  Rows in which more than 512 entries tie at the k-th value, a row
// masked by the type's lowest value with fewer than k columns left among them, cost far more: see select_top.
#include "logits.h"

namespace ddm {
namespace logits {

constexpr int kListCap = 512;        // candidates a selection keeps in LDS

struct ScoreArgs {
    const char* x;
    int64_t n, v, ld_bytes;
    const void* target;
    int target_wide;
    float temperature;
    int top, parts, turns;
    float *logprob, *entropy, *stats, *top_logprob;
    int32_t *rank, *top_index;
    uint8_t* err;
    float4* part_sum;        // [n][parts] m, s, u, rank count as bits
    uint64_t* part_top;      // [n][parts][top] (key << 32) | ~column, 0: none
};

// ---- the k largest of a workgroup's entries ----------------------------------------------------
// A lane's largest entry is a lower bound with a witness of its own, so the k-th largest of the
// lanes' bounds the k-th largest entry from below (tau).  Lanes whose largest reaches tau (little
// more than k of them) have their entries read again, those that reach tau go to LDS and are
// ordered by counting.  More of them than the list holds (rows of equal values) are cut exactly
// by bisection, over entries read again each time, up to 66 times: bounded, but slow.  64 x 32768 bf16 with 20
// alternatives 23 us; constant rows 162; five columns above the type's lowest value 165 (above -inf 23).  4096
// x 131072 with five above the lowest 30.8 ms instead of 0.25.
struct SelectLds {
    uint64_t list[kListCap];
    uint32_t keys[256], hits[kListCap];
    uint32_t tau, n, nhits, sum[4];
};

// One wave: the k-th largest (k at most 64, so at most NT) of NT keys in LDS (kKeyNegInf + 1 if fewer than k are above
// kKeyNegInf).  Bits from the first one in which they differ, a ballot each; once exactly k
// remain, the prefix itself will do.
template <int NT>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t* keys, int k) {
    constexpr int N = NT / 64;
    uint32_t key[N], all = 0xffffffffu, some = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        key[i] = keys[(threadIdx.x & 63) + 64 * i];
        all &= key[i];
        some |= key[i];
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        all &= __shfl_xor(all, d);
        some |= __shfl_xor(some, d);
    }
    const uint32_t differ = __builtin_amdgcn_readfirstlane(all ^ some);
    uint32_t prefix = __builtin_amdgcn_readfirstlane(all);
    if (differ) prefix &= ~((2u << (31 - __builtin_clz(differ))) - 1u);
    for (uint32_t bit = differ ? 1u << (31 - __builtin_clz(differ)) : 0u; bit; bit >>= 1) {
        const uint32_t t = prefix | bit;
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(key[i] >= t));
        if (c >= k) {
            prefix = t;
            if (c == k) break;
        }
    }
    return max(prefix, kKeyNegInf + 1);
}

template <int NT>
__device__ __forceinline__ uint32_t block_sum(uint32_t v, SelectLds& l) {
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) v += __shfl_xor(v, k);
    if (NT == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) l.sum[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t t = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) t += l.sum[w];
    return t;
}

__device__ __forceinline__ void keep(SelectLds& l, uint32_t key, uint32_t col) {
    const uint32_t at = atomicAdd(&l.n, 1u);
    if (at < (uint32_t)kListCap) l.list[at] = ((uint64_t)key << 32) | (uint32_t)~col;
}

// best: the lane's largest key.  hits(tau, add): add(h) for what of the lane's reaches tau, a
// number under 2^32 each; entries(h): how many entries one has, entry(h, i, fn): fn(key, column) of
// the i-th, where there is one; each(fn): fn(key, column) for every entry of the lane.  out(rank,
// packed) for rank 0..k-1.
template <int NT, class Hits, class Entry, class Each, class Out>
__device__ __forceinline__ void select_top(SelectLds& l, uint32_t best, int k, int entries, Hits hits, Entry entry,
                                           Each each, Out out) {
    __syncthreads();
    l.keys[threadIdx.x] = best;
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint32_t t = kth_largest<NT>(l.keys, k);
        if (threadIdx.x == 0) {
            l.tau = t;
            l.n = 0;
            l.nhits = 0;
        }
    }
    __syncthreads();
    const uint32_t tau = l.tau;
    if (best >= tau)
        hits(tau, [&](uint32_t h) {
            const uint32_t at = atomicAdd(&l.nhits, 1u);
            if (at < (uint32_t)kListCap) l.hits[at] = h;
        });
    __syncthreads();
    const uint32_t nhits = l.nhits;
    if (nhits <= (uint32_t)kListCap)
        for (uint32_t i = threadIdx.x; i < nhits * (uint32_t)entries; i += NT)
            entry(l.hits[i / (uint32_t)entries], (int)(i % (uint32_t)entries), [&](uint32_t key, uint32_t col) {
                if (key >= tau) keep(l, key, col);
            });
    __syncthreads();
    uint32_t n = l.n;
    if (n > (uint32_t)kListCap || nhits > (uint32_t)kListCap) {
        // the k-th value exactly (32 halvings), then how far its ties reach (32 more)
        uint32_t lo = tau, hi = 0xffffffffu;            // count(>= lo) >= k, and > hi holds none
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            uint32_t c = 0;
            each([&](uint32_t key, uint32_t) { c += key >= mid; });
            if (block_sum<NT>(c, l) >= (uint32_t)k)
                lo = mid;
            else
                hi = mid - 1;
        }
        const uint32_t kth = lo;
        uint32_t more = 0;
        each([&](uint32_t key, uint32_t) { more += key > kth; });
        const uint32_t ties = (uint32_t)k - block_sum<NT>(more, l);
        uint32_t a = 0, b = 0xffffffffu;                // the lowest column with `ties` ties up to it
        while (a < b) {
            const uint32_t mid = a + (b - a) / 2;
            uint32_t c = 0;
            each([&](uint32_t key, uint32_t col) { c += key == kth && col <= mid; });
            if (block_sum<NT>(c, l) >= ties)
                b = mid;
            else
                a = mid + 1;
        }
        __syncthreads();
        if (threadIdx.x == 0) l.n = 0;
        __syncthreads();
        each([&](uint32_t key, uint32_t col) {
            if (key > kth || (key == kth && col <= a)) keep(l, key, col);
        });
        __syncthreads();
        n = min(l.n, (uint32_t)kListCap);
    }
    for (uint32_t i = threadIdx.x; i < n; i += NT) {
        const uint64_t me = l.list[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += l.list[j] > me;
        if (rank < (uint32_t)k) out((int)rank, me);
    }
    for (uint32_t i = n + threadIdx.x; i < (uint32_t)k; i += NT) out((int)i, 0ull);
}

// ---- one row's results -------------------------------------------------------------------------
// What is common to a row: its reference (see Part), log S (0 for a row with nothing left, NaN for a row
// with NaN or +inf in it).
struct RowLog {
    float m, log_s;
    bool bad, alive;
};
__device__ __forceinline__ RowLog row_log(const Part& p) {
    RowLog r;
    r.m = p.m;
    r.bad = p.s != p.s;
    r.alive = p.s > 0.0f;
    r.log_s = r.alive ? __builtin_amdgcn_logf(p.s) * kLn2 : 0.0f;
    return r;
}

// One thread writes the row's numbers; `ahead` counts the entries before the target's place.
template <typename T>
__device__ __forceinline__ void write_row(const ScoreArgs& a, int64_t r, const Part& p, uint32_t ahead) {
    const RowLog g = row_log(p);
    const float nan = __builtin_nanf("");
    const int64_t t = target_at(a.target, a.target_wide, r);
    const bool counts = t >= 0 && t < a.v;
    float lp = 0.0f;
    int32_t rank = -1;
    uint8_t err = 0;
    if (counts && g.bad) {
        lp = nan;
        err = 1;
    } else if (counts) {
        const float xt = T::one(a.x + r * a.ld_bytes + t * T::kSize);
        lp = xt > -INFINITY ? (xt - g.m) / a.temperature - g.log_s : xt;
        rank = (int32_t)(ahead + (xt > -INFINITY ? 0u : (uint32_t)t));
        err = rank > 0 || !(xt > -INFINITY);
    }
    a.logprob[r] = lp;
    a.entropy[r] = g.bad ? nan : g.alive ? fmaxf(g.log_s - p.u / p.s * kLn2, 0.0f) : 0.0f;
    a.rank[r] = rank;
    a.err[r] = err;
    a.stats[2 * r] = g.m;
    a.stats[2 * r + 1] = g.bad ? nan : g.alive ? __builtin_amdgcn_logf(p.s) : -INFINITY;
    if (r == a.n - 1)                                  // the scans read whole 16-byte words
        for (int64_t i = a.n; i < (a.n + 15) / 16 * 16; ++i) a.err[i] = 0;
}

__device__ __forceinline__ void write_top(const ScoreArgs& a, int64_t r, const RowLog& g, int k, uint64_t packed) {
    const bool some = packed != 0 && !g.bad;
    const float x = of_key((uint32_t)(packed >> 32));
    a.top_index[r * a.top + k] = some ? (int32_t)~(uint32_t)packed : -1;
    a.top_logprob[r * a.top + k] =
        g.bad ? __builtin_nanf("") : some ? (x - g.m) / a.temperature - g.log_s : -INFINITY;
}

// ---- a part of a row ---------------------------------------------------------------------------
template <typename T, int NT, int NV, bool TOP>
__global__ __launch_bounds__(NT) void k_score_parts(ScoreArgs a) {
    __shared__ SelectLds sel;
    __shared__ Part sh_part[NT / 64];
    __shared__ uint32_t sh_ahead[NT / 64];
    extern __shared__ uint32_t turn_best[];              // [turns][NT] the lanes' largest of each turn
    const int64_t r = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x % a.parts);
    const Row<T> row(a.x + r * a.ld_bytes, a.v);
    const int turns = a.turns, j0 = part * NT * NV * turns;

    uint4 raw[NV];
    load_part<T, NT, NV>(row, j0, raw);                  // under way while the target is looked up
    const float c = kLog2e / a.temperature;
    const int64_t t = target_at(a.target, a.target_wide, r);
    const bool counts = t >= 0 && t < a.v;
    const int t32 = counts ? (int)t : -1;
    const float xt = counts ? row.at(t32) : 0.0f;
    // entries before the target's column are ahead of it at equal value; a masked target has
    // every column before it ahead (added with the row) and the alive ones after it
    const float thr_after = counts ? xt : INFINITY;
    const float thr_before = counts && xt > -INFINITY ? below(xt) : INFINITY;

    Lane sums = no_lane();
    float best = -INFINITY;
    uint32_t ahead = 0;
    for (int turn = 0; turn < turns; ++turn) {
        const int jt = j0 + turn * NT * NV;
        if (turn) load_part<T, NT, NV>(row, jt, raw);
        float turn_most = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float f[T::kVec];
            unpack(raw[i], f, T());
            const float most = largest(f);
            turn_most = fmaxf(turn_most, most);
            add_vector<true>(sums, f, most, c);
            const float thr =
                row.col(jt + i * NT + (int)threadIdx.x) + (T::kVec - 1) < t32 ? thr_before : thr_after;
            if (__any(most > thr)) {
#pragma unroll
                for (int e = 0; e < T::kVec; ++e) ahead += (uint32_t)__popcll(__ballot(f[e] > thr));
            }
        }
        best = fmaxf(best, turn_most);
        if (TOP) turn_best[turn * NT + threadIdx.x] = key_of(turn_most);
    }
    if (threadIdx.x == 0 && counts) {                    // the entries before it in its own vector
        const int jt = row.vector_of(t32);
        if (jt >= j0 && jt < j0 + NT * NV * turns)
            for (int i = max(row.col(jt), 0); i < t32; ++i)
                ahead += xt > -INFINITY ? (uint32_t)(row.at(i) == xt) : -(uint32_t)(row.at(i) > xt);
    }
    if ((threadIdx.x & 63) == 0) sh_ahead[threadIdx.x >> 6] = ahead;
    const Part p = block_merge<NT>(part_of(sums, c), c, sh_part);
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < NT / 64; ++w) ahead += sh_ahead[w];
        if (a.parts == 1)
            write_row<T>(a, r, p, ahead);
        else
            a.part_sum[r * a.parts + part] = make_float4(p.m, p.s, p.u, __uint_as_float(ahead));
    }
    if (!TOP) return;
    const RowLog g = row_log(p);
    // a hit is a lane's turn; its entries are read again, as single ones
    auto column = [&](uint32_t turn, uint32_t lane, int i) {
        return row.col(j0 + (int)(turn * NT * NV + lane) + i / T::kVec * NT) + i % T::kVec;
    };
    select_top<NT>(
        sel, key_of(best), a.top, NV * T::kVec,
        [&](uint32_t tau, auto add) {
            for (int turn = 0; turn < turns; ++turn)
                if (turn_best[turn * NT + threadIdx.x] >= tau) add((uint32_t)turn << 8 | threadIdx.x);
        },
        [&](uint32_t h, int i, auto fn) {
            const int col = column(h >> 8, h & 255u, i);
            if (col >= 0 && col < row.v) fn(key_of(row.at(col)), (uint32_t)col);
        },
        [&](auto fn) {
            for (int turn = 0; turn < turns; ++turn)
                for (int i = 0; i < NV * T::kVec; ++i) {
                    const int col = column(turn, threadIdx.x, i);
                    if (col >= 0 && col < row.v) fn(key_of(row.at(col)), (uint32_t)col);
                }
        },
        [&](int k, uint64_t packed) {
            if (a.parts == 1)
                write_top(a, r, g, k, packed);
            else
                a.part_top[(r * a.parts + part) * a.top + k] = packed;
        });
}

// ---- the parts of a row joined -------------------------------------------------------------------
template <typename T, int NT, bool TOP>
__global__ __launch_bounds__(NT) void k_score_join(ScoreArgs a) {
    __shared__ SelectLds sel;
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x & 63;
    const float c = kLog2e / a.temperature;
    Part p = no_part();
    uint32_t ahead = 0;
    for (int i = lane; i < a.parts; i += 64) {         // every wave for itself
        const float4 q = a.part_sum[r * a.parts + i];
        p = merge(p, Part{q.x, q.y, q.z}, c);
        ahead += __float_as_uint(q.w);
    }
    p = wave_merge(p, c);
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) ahead += __shfl_xor(ahead, k);
    if (threadIdx.x == 0) write_row<T>(a, r, p, ahead);
    if (!TOP) return;
    const RowLog g = row_log(p);
    const int n = a.parts * a.top;
    const uint64_t* from = a.part_top + r * n;
    uint32_t best = 0;
    for (int i = threadIdx.x; i < n; i += NT) best = max(best, (uint32_t)(from[i] >> 32));
    auto each = [&](auto fn) {
        for (int i = threadIdx.x; i < n; i += NT) fn((uint32_t)(from[i] >> 32), ~(uint32_t)from[i]);
    };
    select_top<NT>(
        sel, best, a.top, 1,
        [&](uint32_t tau, auto add) {
            for (int i = threadIdx.x; i < n; i += NT)
                if ((uint32_t)(from[i] >> 32) >= tau) add((uint32_t)i);
        },
        [&](uint32_t h, int, auto fn) { fn((uint32_t)(from[h] >> 32), ~(uint32_t)from[h]); }, each,
        [&](int k, uint64_t packed) { write_top(a, r, g, k, packed); });
}

// ---- gradient ------------------------------------------------------------------------------------
// dx_i = (-p_i (A + B log p_i) + [i = t] g_lp + [i = index_k] g_top,k) / T with
// A = g_lp + sum g_top + g_H H, B = g_H: elementwise from the forward's statistics, reading and
// writing every logit once.  The few columns with a term of their own are written again after
// the rest of their part, in full, by one lane each.  Bound by that traffic: 4096 x 65536 bf16 in
// 173 us, 6.2 TB/s, the logits partly still in the last cache from the forward.
struct GradArgs {
    const char* x;
    int64_t n, v, ld_bytes, out_ld_bytes;
    const void* target;
    int target_wide;
    float temperature;
    int top, parts;
    const float *stats, *entropy;
    const int32_t* top_index;
    const float *d_logprob, *d_entropy, *d_top;
    char* out;
};

template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void k_score_grad(GradArgs a) {
    const int64_t r = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x % a.parts);
    const Row<T> row(a.x + r * a.ld_bytes, a.v);
    char* out = a.out + r * a.out_ld_bytes;
    const int j0 = part * NT * NV;
    uint4 raw[NV];
    load_part<T, NT, NV>(row, j0, raw);
    const int lane = threadIdx.x & 63;
    const float m = a.stats[2 * r], log2_s = a.stats[2 * r + 1];
    const float c = kLog2e / a.temperature, inv_t = 1.0f / a.temperature;
    const int64_t t = target_at(a.target, a.target_wide, r);
    const bool counts = t >= 0 && t < a.v;
    const float g_lp = counts && a.d_logprob ? a.d_logprob[r] : 0.0f;
    const float g_h = a.d_entropy ? a.d_entropy[r] : 0.0f;
    int32_t index = -1;
    float g_top = 0.0f;
    if (lane < a.top) {
        index = a.top_index[r * a.top + lane];
        if (index >= a.v) index = -1;                  // the caller's, not read from this call
        if (index >= 0) g_top = a.d_top[r * a.top + lane];
    }
    float all_top = g_top;
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) all_top += __shfl_xor(all_top, k);
    const float A = -(g_lp + all_top + g_h * a.entropy[r]) * inv_t, B = -g_h * kLn2 * inv_t;
    const bool dead = log2_s == -INFINITY;              // nothing left: no gradient
    // the columns with a term of their own, read before any store: out may be the logits
    auto mine = [&](int col) {
        const int j = row.vector_of(col);
        return j >= j0 && j < j0 + NT * NV;
    };
    const bool first = threadIdx.x < 64;
    const bool put_top = first && index >= 0 && mine(index);
    const bool put_t = threadIdx.x == 0 && counts && mine((int)t);
    const float x_top = put_top ? row.at(index) : 0.0f, x_t = put_t ? row.at((int)t) : 0.0f;
    __syncthreads();
    auto value = [&](float x) {
        const float d = (x - m) * c - log2_s;
        return dead ? 0.0f : __builtin_amdgcn_exp2f(d) * fmaf(B, fmaxf(d, kDead), A);
    };
    store_part<T, NT, NV>(
        row, out, j0,
        [&](int i, float (&f)[T::kVec]) {
            unpack(raw[i], f, T());
#pragma unroll
            for (int e = 0; e < T::kVec; ++e) f[e] = value(f[e]);
        },
        [](int) { return 0u; });
    __syncthreads();
    auto put = [&](int col, float x, float extra) {
        T::store(out + col * T::kSize, dead ? 0.0f : fmaf(extra, inv_t, value(x)));
    };
    const bool listed = __any(counts && index == t);
    if (put_top) put(index, x_top, g_top + (counts && index == t ? g_lp : 0.0f));
    if (put_t && !listed) put((int)t, x_t, g_lp);
}

// ---- launch shapes ---------------------------------------------------------------------------------
// One wave a row while the row fits its registers (512 vectors of 16 bytes); longer rows in
// parts of 256 lanes, 8 vectors a lane and turn, with as many turns (a selection a part) or as
// few vectors as leave workgroups enough to fill 256 CUs several times over.
inline Shape shape_of(int64_t n, int64_t nvec, bool turns) {
    Shape s{256, 8, 1, 1};
    if (nvec <= 64 * 8) {
        s.nt = 64;
        s.nv = nvec <= 64 ? 1 : nvec <= 128 ? 2 : nvec <= 256 ? 4 : 8;
    } else {
        while (s.nv > 1 && n * ceil_div(nvec, 256 * s.nv) < 1024 && ceil_div(nvec, 128 * s.nv) <= kMaxParts) s.nv /= 2;
        while (turns && s.turns < 4 && n * ceil_div(nvec, 256 * s.nv * s.turns * 2) >= 8192) s.turns *= 2;
    }
    s.parts = (int)ceil_div(nvec, (int64_t)s.nt * s.nv * s.turns);
    return s;
}
inline int64_t score_scratch(const Shape& s, int64_t n, int64_t top) {
    return s.parts == 1 ? 0 : n * s.parts * (16 + 8 * top);
}

}  // namespace logits
}  // namespace ddm

using namespace ddm;
using namespace ddm::logits;

extern "C" int64_t ddm_token_scores_scratch_bytes(int64_t n, int64_t v, int32_t dtype, int32_t top) {
    if (n <= 0 || v < 1 || v > kMaxColumns || top < 0 || top > kMaxTop) return 0;
    const int vec = dtype == DDM_F32 ? 4 : 8;            // whether rows start aligned or not
    const int64_t a = score_scratch(shape_of(n, ceil_div(v, vec), true), n, top);
    const int64_t b = score_scratch(shape_of(n, ceil_div(v + vec - 1, vec), true), n, top);
    return a > b ? a : b;
}

extern "C" int ddm_token_scores(const void* logits, int32_t dtype, int64_t n, int64_t v, int64_t ld,
                                const void* target, int32_t target_bytes, float temperature, int32_t top,
                                float* logprob, float* entropy, float* stats, int32_t* rank, uint8_t* err,
                                float* top_logprob, int32_t* top_index, void* scratch, ddm_stream_t stream,
                                ddm_event_t ev_begin, ddm_event_t ev_end) {
    if (int rc = check_rows("ddm_token_scores", dtype, n, v, ld, target_bytes, temperature, top)) return rc;
    if (n == 0) return timed_nothing(ev_begin, ev_end, stream);
    const int size = dtype == DDM_F32 ? 4 : 2;
    const Shape s = shape_of(n, vectors_of(logits, ld * size, v, 16 / size), true);
    if (int rc = check_grid("ddm_token_scores", n * s.parts, s.nt)) return rc;
    if (!logits || !target || !logprob || !entropy || !stats || !rank || !err || (top && (!top_logprob || !top_index)) ||
        (s.parts > 1 && !scratch)) {
        set_error("ddm_token_scores: invalid argument (null pointer)");
        return DDM_E_ARG;
    }
    const hipStream_t st = as_hip(stream);
    return timed(ev_begin, ev_end, st, [&] {
        return with_type(dtype, [&](auto type) {
            using T = decltype(type);
            ScoreArgs a{(const char*)logits, n, v, ld * T::kSize, target, target_bytes == 8, temperature, top, s.parts,
                        s.turns, logprob, entropy, stats, top_logprob, rank, top_index, err, (float4*)scratch,
                        (uint64_t*)((char*)scratch + n * s.parts * 16)};
            with_part_shape(s, [&](auto nt, auto nv) {
                if (top)
                    k_score_parts<T, nt(), nv(), true><<<dim3((unsigned)(n * s.parts)), nt(), nt() * s.turns * 4, st>>>(a);
                else
                    k_score_parts<T, nt(), nv(), false><<<dim3((unsigned)(n * s.parts)), nt(), 0, st>>>(a);
            });
            if (int rc = launch_status("ddm_token_scores")) return rc;
            if (s.parts > 1) {
                if (!top)
                    k_score_join<T, 64, false><<<dim3((unsigned)n), 64, 0, st>>>(a);
                else if (s.parts * top <= 512)                 // 8 a lane: a wave is enough
                    k_score_join<T, 64, true><<<dim3((unsigned)n), 64, 0, st>>>(a);
                else
                    k_score_join<T, 256, true><<<dim3((unsigned)n), 256, 0, st>>>(a);
            }
            return launch_status("ddm_token_scores");
        });
    });
}

extern "C" int ddm_token_scores_grad(const void* logits, int32_t dtype, int64_t n, int64_t v, int64_t ld,
                                     const void* target, int32_t target_bytes, float temperature, int32_t top,
                                     const float* stats, const float* entropy, const int32_t* top_index,
                                     const float* d_logprob, const float* d_entropy, const float* d_top, void* out,
                                     int64_t out_ld, ddm_stream_t stream, ddm_event_t ev_begin, ddm_event_t ev_end) {
    if (int rc = check_rows("ddm_token_scores_grad", dtype, n, v, ld, target_bytes, temperature, top)) return rc;
    if (n == 0) return timed_nothing(ev_begin, ev_end, stream);
    if (!logits || !target || !stats || !entropy || !out || out_ld < v || (top && (!top_index || !d_top))) {
        set_error("ddm_token_scores_grad: invalid argument (null pointer or output stride)");
        return DDM_E_ARG;
    }
    const int size = dtype == DDM_F32 ? 4 : 2;
    const Shape s = shape_of(n, vectors_of(logits, ld * size, v, 16 / size), false);
    if (int rc = check_grid("ddm_token_scores_grad", n * s.parts, s.nt)) return rc;
    const hipStream_t st = as_hip(stream);
    return timed(ev_begin, ev_end, st, [&] {
        return with_type(dtype, [&](auto type) {
            using T = decltype(type);
            GradArgs a{(const char*)logits, n, v, ld * T::kSize, out_ld * T::kSize, target, target_bytes == 8,
                       temperature, top, s.parts, stats, entropy, top_index, d_logprob, d_entropy, d_top, (char*)out};
            with_part_shape(s, [&](auto nt, auto nv) {
                k_score_grad<T, nt(), nv()><<<dim3((unsigned)(n * s.parts)), nt(), 0, st>>>(a);
            });
            return launch_status("ddm_token_scores_grad");
        });
    });
}
