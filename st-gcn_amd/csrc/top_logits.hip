// The largest k scores of every row, with their classes, and the log of what the other classes weigh together.
//
// Classes are ordered by (score descending, class ascending); NaN comes first.  rest = log sum over the unlisted
// classes of e^{x/T}, summed over them alone (never as a difference of sums).
//
// One pass over the scores.  A workgroup walks its row (or its piece of one) in batches and keeps, in LDS, every score
// that may still be among the k first: those beyond `tau`, a bound that k scores are known to reach.  The first bound
// comes from the first batch: k of its threads' (or vectors') maxima reach it, so about k to 2k of the batch's scores
// do.  When more than a few k have gathered, the k-th of them becomes the bound.  A score that is not kept, or is dropped
// from the buffer, enters the sum of the rest at once, under a running maximum, so nothing is read twice.
#include "scores.h"

namespace {

constexpr int MAX_K = 256;
constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.6931471805599453094;
typedef unsigned long long u64;

// position in the order as one number: larger is earlier
__device__ __forceinline__ u64 place(uint32_t key, int j) { return ((u64)key << 32) | (uint32_t)~j; }
__device__ __forceinline__ int place_class(u64 p) { return (int)~(uint32_t)p; }

// Sum of 2^{x c} under a running maximum.
struct RestSum {
    float m = -INFINITY, s = 0.f;
    __device__ __forceinline__ void raise(float to, float c) {
        if (to > m) { s *= m == -INFINITY ? 0.f : exp2_32((m - to) * c); m = to; }
    }
    __device__ __forceinline__ void add(float x, float c) { s += exp2_32((x - (m == -INFINITY ? 0.f : m)) * c); }   // x <= m, or all are -inf
    __device__ __forceinline__ void take(float x, float c) {
        raise(x, c);
        s += x == m ? (m == -INFINITY ? 0.f : 1.f) : exp2_32((x - m) * c);
    }
};

template <int W> __device__ __forceinline__ void group_sync() {
    if constexpr (W == 1) { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier(); }
    else lds_barrier();                            // LDS only: loads of the next batch stay in flight
}

// Buffer of candidates of a group of W waves.
template <int W> struct Shared {
    static constexpr int CAP = W == 1 ? 512 : 2048;
    u64 cand[CAP];
    u64 kept[MAX_K];
    uint32_t maxima[W == 1 ? 64 : 1024];
    u64 tau;
    int count, missed, nkept;
    float rm[4]; double rs[4];
};

// The k-th largest of `c` (> k) distinct places, by one wave: bisection of the key, then of the class among equal keys.
// With at most 512 of them their keys stay in registers.
__device__ __forceinline__ u64 kth_place(const u64* cand, int c, int k) {
    const int lane = threadIdx.x & 63;
    uint32_t v = 0;
    if (c <= 512) {
        uint32_t key[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) key[i] = lane + 64 * i < c ? (uint32_t)(cand[lane + 64 * i] >> 32) : 0;
        for (int b = 31; b >= 0; --b) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) if (64 * i < c) n += __popcll(__ballot(key[i] >= (v | 1u << b)));
            if (n >= k) v |= 1u << b;
        }
    } else {
        for (int b = 31; b >= 0; --b) {
            int n = 0;
            for (int i = lane; i - lane < c; i += 64) n += __popcll(__ballot(i < c && (uint32_t)(cand[i < c ? i : 0] >> 32) >= (v | 1u << b)));
            if (n >= k) v |= 1u << b;
        }
    }
    int above = 0, equal = 0;
    for (int i = lane; i - lane < c; i += 64) {
        const uint32_t key = i < c ? (uint32_t)(cand[i] >> 32) : 0;
        above += __popcll(__ballot(i < c && key > v));
        equal += __popcll(__ballot(i < c && key == v));
    }
    if (above + equal == k) return (u64)v << 32;
    uint32_t l = 0;
    for (int b = 31; b >= 0; --b) {
        int n = above;
        for (int i = lane; i - lane < c; i += 64) {
            const u64 p = i < c ? cand[i] : 0;
            n += __popcll(__ballot(i < c && (uint32_t)(p >> 32) == v && (uint32_t)p >= (l | 1u << b)));
        }
        if (n >= k) l |= 1u << b;
    }
    return (u64)v << 32 | l;
}

// Keeps the k first of the buffer's entries; the others go to the rest.  tau = the k-th.
template <int W> __device__ __forceinline__ void compact(Shared<W>& sh, int tid, int k, RestSum& rest, float c) {
    constexpr int G = W * 64, CAP = Shared<W>::CAP;
    group_sync<W>();
    const int n = min(sh.count, CAP);
    if (n <= k) return;                            // the same in every thread
    if (tid < 64) {
        const u64 t = kth_place(sh.cand, n, k);
        if (tid == 0) { sh.tau = t; sh.nkept = 0; }
    }
    group_sync<W>();
    const u64 t = sh.tau;
    for (int i = tid; i < n; i += G) {
        const u64 p = sh.cand[i];
        if (p >= t) sh.kept[atomicAdd(&sh.nkept, 1)] = p;
        else if (p) rest.take(key_score((uint32_t)(p >> 32)), c);
    }
    group_sync<W>();
    for (int i = tid; i < k; i += G) sh.cand[i] = sh.kept[i];
    if (tid == 0) sh.count = k;
    group_sync<W>();
}

// Offers this thread's pending scores (bit e of `pending`: x(e), class(e)) to the buffer until all of the group's are kept
// or beyond the bound.  Returns the bits of the scores that are kept.
template <int W, typename X, typename J>
__device__ __forceinline__ u64 offer(Shared<W>& sh, int tid, int k, u64 pending, X x, J cls, RestSum& rest, float c) {
    constexpr int CAP = Shared<W>::CAP;
    u64 kept = 0;
    for (;;) {
        int n = 0, base = 0;
        if (pending) {
            n = __popcll(pending);
            base = atomicAdd(&sh.count, n);
            if (base + n <= CAP) {
                for (u64 q = pending; q; q &= q - 1) {
                    const int e = __ffsll(q) - 1;
                    sh.cand[base++] = place(score_key(x(e)), cls(e));
                }
                kept |= pending;
                pending = 0;
            } else {
                for (; base < CAP; ++base) sh.cand[base] = 0;
                sh.missed = 1;
            }
        }
        group_sync<W>();
        const int count = sh.count, missed = sh.missed;
        group_sync<W>();
        if (!missed && count <= (CAP / 4 > 3 * k ? CAP / 4 : 3 * k)) return kept;
        if (tid == 0) sh.missed = 0;
        compact<W>(sh, tid, k, rest, c);
        if (!missed) return kept;
        const u64 t = sh.tau;
        u64 left = 0;
        for (u64 q = pending; q; q &= q - 1) {
            const int e = __ffsll(q) - 1;
            if (place(score_key(x(e)), cls(e)) > t) left |= q & -q;    // else it stays where it is and is summed as rest
        }
        pending = left;
    }
}

// Piece `piece` (of `pieces`) of row r.  With one piece the answer is written; else its k places, its rest's maximum and sum.
struct TopArgs {
    const void* x; size_t stride; int rows, n, k, pieces;
    float c; double T;
    float* values; long long* indices; float* rest;
    u64* part; float2* part_rest;                  // [rows][pieces][k], [rows][pieces]
};

template <typename T, int W>
__device__ void slow_row(const T* x, int lo, int hi, int tid, int k, Shared<W>& sh, RestSum& rest, float c) {
    // scores that are NaN, or more infinities than k: the k first one after the other, then the rest in two passes
    constexpr int G = W * 64;
    u64 last = ~0ull;
    __shared__ u64 red[4];
    for (int q = 0; q < k; ++q) {
        u64 best = 0;
        for (int j = lo + tid; j < hi; j += G) {
            const u64 p = place(score_key(load_elem(x, j)), j);
            if (p > best && (q == 0 || p < last)) best = p;
        }
        best = wave_reduce(best, OpMax());
        if constexpr (W > 1) {
            __syncthreads();
            if ((tid & 63) == 0) red[tid >> 6] = best;
            __syncthreads();
            for (int w = 0; w < W; ++w) best = red[w] > best ? red[w] : best;
        }
        last = best;
        if (tid == 0) sh.cand[q] = best;           // 0: fewer scores than k in this piece
    }
    rest = RestSum();
    for (int j = lo + tid; j < hi; j += G) {
        const float v = load_elem(x, j);
        if (place(score_key(v), j) < last) { if (v != v) rest.s = NAN; else rest.take(v, c); }
    }
    group_sync<W>();
    if (tid == 0) sh.count = k;
    group_sync<W>();
}

// rest of the group: its threads' sums joined.  Every thread gets the pair.
template <int W> __device__ __forceinline__ void join_rest(Shared<W>& sh, int tid, const RestSum& r, float c, float& m, double& s) {
    m = wave_reduce(r.m, OpFMax());
    if constexpr (W > 1) {
        if ((tid & 63) == 0) sh.rm[tid >> 6] = m;
        __syncthreads();
        for (int w = 0; w < W; ++w) m = fmaxf(m, sh.rm[w]);
    }
    s = (double)r.s * (r.m == m || r.m == -INFINITY ? 1.0 : (double)exp2_32((r.m - m) * c));
    s = wave_reduce(s, OpSum());
    if constexpr (W > 1) {
        if ((tid & 63) == 0) sh.rs[tid >> 6] = s;
        __syncthreads();
        s = 0;
        for (int w = 0; w < W; ++w) s += sh.rs[w];
    }
}

// The buffer's k first in order, into the answer.
template <int W> __device__ void write_row(const TopArgs& a, size_t r, Shared<W>& sh, int tid) {
    constexpr int G = W * 64;
    const int k = a.k;
    for (int i = tid; i < k; i += G) {
        const u64 p = sh.cand[i];
        int rank = 0;
        for (int o = 0; o < k; ++o) rank += sh.cand[o] > p ? 1 : 0;
        a.values[r * k + rank] = key_score((uint32_t)(p >> 32));
        a.indices[r * k + rank] = place_class(p);
    }
}

template <typename T, int W>
__global__ __launch_bounds__(256) void top_scan_kernel(TopArgs a) {
    constexpr int VEC = ET<T>::VEC, G = W * 64, NB = 16 / VEC, PER = NB * VEC, ROWS = W == 1 ? 4 : 1;
    __shared__ Shared<W> sh_[ROWS];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, tid = W == 1 ? lane : threadIdx.x;
    const size_t job = W == 1 ? (size_t)blockIdx.x * ROWS + wave : blockIdx.x;
    const size_t r = W == 1 ? job : job / a.pieces;
    if (W == 1 && r >= (size_t)a.rows) return;
    const int piece = W == 1 ? 0 : (int)(job % a.pieces);
    Shared<W>& sh = sh_[W == 1 ? wave : 0];
    const int n = a.n, k = a.k;
    const float c = a.c;
    const T* x = (const T*)((const char*)a.x + r * a.stride * ET<T>::ES);
    const RowSpan<T> sp(x, n);
    // vectors of this piece: whole batches, the row's edges with its first and last piece
    const int batches = (sp.nvec + G * NB - 1) / (G * NB);
    const int b0 = (int)((long long)batches * piece / a.pieces), b1 = (int)((long long)batches * (piece + 1) / a.pieces);
    const bool with_head = piece == 0, with_tail = piece == a.pieces - 1;
    const int v1 = min(b1 * G * NB, sp.nvec);

    if (tid == 0) { sh.count = 0; sh.missed = 0; sh.tau = 0; }
    RestSum rest;
    i32x4 v[NB], nx[NB];
    auto load = [&](int b, i32x4* to) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int at = b * G * NB + i * G + tid;
            if (at < v1) to[i] = load_vec(x, sp.vec_at(at));
            else { const int w = ET<T>::IS_BF16 ? (int)0xFF80FF80u : (int)0xFF800000u; to[i] = i32x4{w, w, w, w}; }
        }
    };
    load(b0, nx);
    const float xh = with_head && tid < sp.head ? load_elem(x, tid) : -INFINITY;

    for (int b = b0; b < b1 || b == b0; ++b) {
#pragma unroll
        for (int i = 0; i < NB; ++i) v[i] = nx[i];
        if (b + 1 < b1) load(b + 1, nx);
        float top = vec_max<T>(v[0]);
#pragma unroll
        for (int i = 1; i < NB; ++i) top = fmaxf(top, vec_max<T>(v[i]));
        if (b == b0) {
            // a bound that k scores of this batch reach, to 16 bits of the key: from 64 W maxima of threads, or 64 W NB of vectors
            const bool fine = W > 1 && k > 64;
            if (fine) {
#pragma unroll
                for (int i = 0; i < NB; ++i) sh.maxima[(i * G + tid) & 1023] = score_key(vec_max<T>(v[i]));
            } else sh.maxima[tid] = score_key(top);
            group_sync<W>();
            if (tid < 64) {
                const int have = fine ? W * NB : W;
                uint32_t m[16], t = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) m[i] = i < have ? sh.maxima[(lane + 64 * i) & (W == 1 ? 63 : 1023)] : 0;
                for (int bit = 31; bit >= 16; --bit) {
                    const uint32_t to = t | 1u << bit;
                    int cnt = 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) if (i < have) cnt += __popcll(__ballot(m[i] >= to));
                    if (cnt >= k) t = to;
                }
                // a bound at or below -inf: everything
                if (lane == 0) sh.tau = t <= KEY_NEG_INF ? 0 : (u64)t << 32;
            }
            group_sync<W>();
        }
        const u64 tau = sh.tau;
        // The first batch's bound is a key that k scores reach; a later batch's classes come after the buffer's, and of
        // those only larger keys than tau's are earlier in the order.
        const uint32_t tk = (uint32_t)(tau >> 32), least = tau == 0 ? 0 : b == b0 ? tk : tk + 1;
        u64 pending = 0;
        if (least == 0 || score_key(top) >= least) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int at = b * G * NB + i * G + tid;
                float f[VEC];
                unpack16<T>(v[i], f);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (at < v1 && score_key(f[j]) >= least) pending |= 1ull << (i * VEC + j);
            }
        }
        if (b == b0 && with_head && tid < sp.head && score_key(xh) >= least) pending |= 1ull << PER;
        auto cls = [&](int e) { return e == PER ? tid : sp.vec_at(b * G * NB + (e / VEC) * G + tid) + e % VEC; };
        const u64 kept = offer<W>(sh, tid, k, pending, [&](int e) { return load_elem(x, cls(e)); }, cls, rest, c);
#pragma unroll
        for (int i = 0; i < NB; ++i) asm volatile("" : "+v"(v[i]));        // unpacked again below rather than held as floats
        if (kept) {
            top = -INFINITY;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                drop_listed<T>(v[i], (uint32_t)(kept >> (i * VEC)) & ((1u << VEC) - 1));
                top = fmaxf(top, vec_max<T>(v[i]));
            }
        }
        rest.raise(top, c);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            float f[VEC];
            unpack16<T>(v[i], f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) rest.add(f[j], c);
        }
        if (b == b0 && with_head && tid < sp.head && !(kept >> PER & 1)) { if (xh != xh) rest.s = NAN; else rest.take(xh, c); }
    }
    if (with_tail) {                               // the classes behind the last whole vector, last in the order of classes
        const int tail = sp.edge - sp.head, j = n - tail + tid;
        const float xt = tid < tail ? load_elem(x, j) : 0.f;
        const u64 kept = offer<W>(sh, tid, k, tid < tail && place(score_key(xt), j) > sh.tau ? 1ull : 0ull, [&](int) { return xt; },
                                  [&](int) { return j; }, rest, c);
        if (tid < tail && !kept) { if (xt != xt) rest.s = NAN; else rest.take(xt, c); }
    }
    compact<W>(sh, tid, k, rest, c);
    bool nan = rest.s != rest.s;
    if constexpr (W == 1) nan = __ballot(nan) != 0; else nan = __syncthreads_or(nan);
    if (nan) {
        const int lo = with_head ? 0 : sp.vec_at(b0 * G * NB), hi = with_tail ? n : sp.vec_at(v1);
        slow_row<T, W>(x, lo, hi, tid, k, sh, rest, c);
    }
    float m; double s;
    join_rest<W>(sh, tid, rest, c, m, s);
    if (a.pieces == 1) {
        write_row<W>(a, r, sh, tid);
        if (tid == 0) a.rest[r] = s != s ? NAN : m == -INFINITY ? -INFINITY : (float)((double)m / a.T + log(s));
    } else {
        const int have = min(sh.count, k);
        for (int i = tid; i < k; i += G) a.part[job * k + i] = i < have ? sh.cand[i] : 0;
        if (tid == 0) a.part_rest[job] = make_float2(m, (float)s);
    }
}

}  // namespace

// Pieces a row is split into: rows fill the chip by themselves from two workgroups a compute unit on; below that a row
// is cut into pieces of at least one batch.
static int top_pieces(int dtype, int rows, int ncls, int k) {
    (void)dtype; (void)rows; (void)ncls; (void)k;
    return 1;
}

extern "C" int stgcn_top_logits(int dtype, const void* logits, size_t row_stride, int rows, int ncls, int k, double temperature,
                                float* values, int64_t* indices, float* rest, void* stream) {
    if (!logits || !values || !indices || !rest || rows < 1 || ncls < 1 || ncls > (1 << 20) || row_stride < (size_t)ncls || k < 1 || k > MAX_K
        || k > ncls || !(temperature > 0.0) || !(temperature < 1e30) || (dtype != STGCN_F32 && dtype != STGCN_BF16)) return STGCN_ERR_ARG;
    TopArgs a = {logits, row_stride, rows, ncls, k, top_pieces(dtype, rows, ncls, k), (float)(LOG2E / temperature), temperature, values, (long long*)indices, rest,
                 nullptr, nullptr};
    const hipStream_t s = (hipStream_t)stream;
    if (ncls <= 512) {
        const unsigned quads = (unsigned)((rows + 3) / 4);
        if (dtype == STGCN_BF16) top_scan_kernel<bf16, 1><<<quads, 256, 0, s>>>(a); else top_scan_kernel<float, 1><<<quads, 256, 0, s>>>(a);
    } else {
        if (dtype == STGCN_BF16) top_scan_kernel<bf16, 4><<<rows, 256, 0, s>>>(a); else top_scan_kernel<float, 4><<<rows, 256, 0, s>>>(a);
    }
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}
