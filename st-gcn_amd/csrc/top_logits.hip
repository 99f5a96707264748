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
//
// Many rows are bound by their instructions: 13 vector instructions a score with k 1 and 20 with k 64, whose issue takes 85 and
// 76 of 100 cycles of every SIMD (4096 x 65536 bf16: 135 and 206 us, 2.6 TB/s with k 64); the rest is what a row costs by
// itself, the first bound and the ranking of the answer.  Few rows are cut into pieces, or one compute unit would read each
// alone (4 x 131071 float32, k 128: 170 us in one piece, 29 in 25, half of it the join).
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

// Buffer of candidates of a group of W waves.  Its order is the same every run (places are dealt by prefix counts, not by
// atomics), and with it the order in which dropped scores are added to the rest.  `add` holds what each wave appends in a
// batch; three sets take turns, so that one barrier a batch is enough: while all read a batch's counts, nobody writes them.
template <int W> struct Shared {
    static constexpr int CAP = W == 1 ? 512 : 2048;
    u64 cand[CAP];
    static constexpr int EQ = W == 1 ? 128 : 1024;
    uint32_t maxima[EQ];                           // of the first batch; later the classes of equal scores
    u64 tau; float lim;                            // the bound; scores x with !(x <= lim) may be earlier in the order
    int add[3][W];
    float rm[4]; double rs[4];
    // A thread's sums of before, in 64 bits, relative to far_m: what a thread adds up in 32 bits is 512 terms at most, and
    // what a compaction drops a lane (one wave's, 64 terms a batch where the scores ascend).  W = 1: rows of 512 classes.
    double far_s[W == 1 ? 1 : W * 64]; float far_m[W == 1 ? 1 : W * 64];
};
constexpr int FLUSH = 32;                          // batches of 16 scores a thread

// 2^{(from - to) c} for a sum relative to `from` (-inf: the sum is 0, or NaN)
__device__ __forceinline__ double rebase(float from, float to, float c) { return from == to || from == -INFINITY ? 1.0 : (double)exp2_32((from - to) * c); }
template <int W> __device__ __forceinline__ void far_clear(Shared<W>& sh, int tid) {
    if constexpr (W > 1) { sh.far_s[tid] = 0; sh.far_m[tid] = -INFINITY; }
}
template <int W> __device__ __forceinline__ void far_add(Shared<W>& sh, int tid, const RestSum& r, float c) {
    const float was = sh.far_m[tid], m = fmaxf(was, r.m);
    sh.far_s[tid] = sh.far_s[tid] * rebase(was, m, c) + (double)r.s * rebase(r.m, m, c);
    sh.far_m[tid] = m;
}
__host__ __device__ __forceinline__ int buffer_limit(int k) { return 2 * k + 64; }       // beyond it the bound is raised

// The largest score before key `k` (> -inf) in the order of the scores.
__device__ __forceinline__ float score_before(uint32_t k) { return key_score(k == 0x80000000u ? 0x7FFFFFFEu : k - 1); }   // -0 is 0

// Bits of a key that carry something: a bf16 score has 16.  long_key gives back the lowest 16, which are the sign's, and those
// of NaN, whose one key is all ones.
template <typename T> constexpr int KEY_SHIFT = ET<T>::IS_BF16 ? 16 : 0;
template <typename T> __device__ __forceinline__ uint32_t short_key(u64 p) { return (uint32_t)(p >> (32 + KEY_SHIFT<T>)); }
template <typename T> __device__ __forceinline__ uint32_t long_key(uint32_t s) {
    return ET<T>::IS_BF16 ? s << 16 | ((s & 0x8000u) && s != KEY_NAN >> 16 ? 0u : 0xFFFFu) : s;
}


// The k-th largest of `c` numbers v(i) (i < c, c >= k) that are not all distinct, by one wave, bit by bit below those that
// all have in common; with at most 512 of them they stay in registers.
template <typename V> __device__ __forceinline__ uint32_t kth_largest(V v, int c, int k) {
    const int lane = threadIdx.x & 63;
    uint32_t r[8], lo = ~0u, hi = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        r[i] = 0;
        if (64 * i < c && lane + 64 * i < c) { r[i] = v(lane + 64 * i); lo = min(lo, r[i]); hi = max(hi, r[i]); }
    }
    for (int i = lane + 512; i < c; i += 64) { const uint32_t s = v(i); lo = min(lo, s); hi = max(hi, s); }
    lo = wave_reduce(lo, [](uint32_t a, uint32_t b) { return min(a, b); });
    hi = wave_reduce(hi, OpMax());
    if (lo == hi) return lo;
    const int first = 31 - __clz(lo ^ hi);
    uint32_t t = first == 31 ? 0 : hi >> (first + 1) << (first + 1);
    for (int b = first; b >= 0; --b) {
        const uint32_t to = t | 1u << b;
        int n = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) if (64 * i < c) n += __popcll(__ballot(r[i] >= to));
        for (int i = lane + 512; i - lane < c; i += 64) n += __popcll(__ballot(i < c && v(i < c ? i : 0) >= to));
        if (n >= k) t = to;
    }
    return t;
}

// The k-th largest of `c` (> k) distinct places, by one wave: the key, then the class among equal keys, which are
// gathered in `equal` (EQ numbers of LDS) first.
template <typename T, int EQ> __device__ __forceinline__ u64 kth_place(const u64* cand, uint32_t* equal, int c, int k) {
    const int lane = threadIdx.x & 63;
    const uint32_t v = kth_largest([&](int i) { return short_key<T>(cand[i]); }, c, k);
    int above = 0, same = 0;
    for (int i = lane; i - lane < c; i += 64) {
        const u64 p = i < c ? cand[i] : 0;
        const uint32_t s = short_key<T>(p);
        const u64 q = __ballot(i < c && s == v);
        above += __popcll(__ballot(i < c && s > v));
        if (i < c && s == v && same + lanes_below(q) < EQ) equal[same + lanes_below(q)] = (uint32_t)p;
        same += __popcll(q);
    }
    const u64 t = (u64)long_key<T>(v) << 32;
    if (above + same == k) return t;
    if (same <= EQ) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
        return t | kth_largest([&](int i) { return equal[i]; }, same, k - above);
    }
    uint32_t l = 0;                                // many equal scores
    for (int b = 31; b >= 0; --b) {
        int n = above;
        for (int i = lane; i - lane < c; i += 64) {
            const u64 p = i < c ? cand[i] : 0;
            n += __popcll(__ballot(i < c && short_key<T>(p) == v && (uint32_t)p >= (l | 1u << b)));
        }
        if (n >= k) l |= 1u << b;
    }
    return t | l;
}

// Keeps the k first of the buffer's n entries, in the order in which they stand; the others go to the rest.  The k-th becomes
// the bound.  One wave's work.
template <typename T, int W> __device__ __forceinline__ void compact(Shared<W>& sh, int tid, int& n, int k, RestSum& rest, float c) {
    group_sync<W>();
    if (n <= k) return;                            // the same in every thread
    if (tid < 64) {
        const u64 t = kth_place<T, Shared<W>::EQ>(sh.cand, sh.maxima, n, k);
        int at = 0;
        RestSum dropped;
        for (int i = 0; i < n; i += 64) {          // entries only move towards the front
            const u64 p = i + tid < n ? sh.cand[i + tid] : 0;
            const u64 keep = __ballot(p >= t && p);
            if (p >= t && p) sh.cand[at + lanes_below(keep)] = p;
            else if (p) { if constexpr (W > 1) dropped.take(key_score((uint32_t)(p >> 32)), c); else rest.take(key_score((uint32_t)(p >> 32)), c); }
            at += __popcll(keep);
        }
        if constexpr (W > 1) far_add<W>(sh, tid, dropped, c);
        if (tid == 0) { sh.tau = t; sh.lim = key_score((uint32_t)(t >> 32)); }
    }
    n = k;
    group_sync<W>();
}

// A key, to 16 bits, that k of the first 64 `some` (<= 64 MOST) maxima reach; by one wave.  0: not that many are there.
template <int MOST> __device__ __forceinline__ uint32_t bound_of_maxima(const uint32_t* maxima, int some, int k) {
    const int lane = threadIdx.x & 63;
    uint32_t m[MOST], t = 0;
#pragma unroll
    for (int i = 0; i < MOST; ++i) m[i] = i < some ? maxima[lane + 64 * i] : 0;
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t to = t | 1u << bit;
        int cnt = 0;
#pragma unroll
        for (int i = 0; i < MOST; ++i) if (i < some) cnt += __popcll(__ballot(m[i] >= to));
        if (cnt >= k) t = to;
    }
    return t;
}

// What the waves append in a batch: `mine` entries of this wave; returns this wave's first slot, n becomes the new count
// (which may be beyond CAP).
template <int W> __device__ __forceinline__ int deal_slots(Shared<W>& sh, int tid, int& n, int& turn, int mine) {
    int slot = n;
    if constexpr (W == 1) { n += mine; return slot; }
    const int wave = tid >> 6;
    if ((tid & 63) == 0) sh.add[turn][wave] = mine;
    group_sync<W>();
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int s = __builtin_amdgcn_readfirstlane(sh.add[turn][w]);
        if (w < wave) slot += s;
        n += s;
    }
    turn = turn == 2 ? 0 : turn + 1;
    return slot;
}

// Appends this thread's pending scores (bit e: the score x(e) of class cls(e)), however many there are: what finds no
// room is held against the raised bound and offered again.  Returns the bits that are kept; the others belong to the rest.
// The way of row ends and of full buffers.
template <typename T, int W, typename X, typename J>
__device__ __forceinline__ uint32_t offer(Shared<W>& sh, int tid, int& n, int& turn, int k, uint32_t pending, X x, J cls, RestSum& rest, float c) {
    constexpr int CAP = Shared<W>::CAP;
    uint32_t kept = 0;
    for (;;) {
        const int m = __popc(pending);
        int below = 0, all = 0;
#pragma unroll
        for (int b = 0; b < 6; ++b) {
            const u64 q = __ballot(m >> b & 1);
            below += lanes_below(q) << b;
            all += __popcll(q) << b;
        }
        int slot = deal_slots<W>(sh, tid, n, turn, all) + below;
        const bool full = n > CAP;
        if (pending) {
            if (slot + m <= CAP) {
                for (uint32_t q = pending; q; q &= q - 1) { const int e = __ffs(q) - 1; sh.cand[slot++] = place(score_key(x(e)), cls(e)); }
                kept |= pending;
                pending = 0;
            } else for (; slot < CAP; ++slot) sh.cand[slot] = 0;
        }
        if (full) n = CAP;
        if (!full && n <= buffer_limit(k)) return kept;
        compact<T, W>(sh, tid, n, k, rest, c);
        if (!full) return kept;
        uint32_t left = 0;
        for (uint32_t q = pending; q; q &= q - 1) { const int e = __ffs(q) - 1; if (place(score_key(x(e)), cls(e)) > sh.tau) left |= q & -q; }
        pending = left;
    }
}

// Piece `piece` (of `pieces`) of row r.  With one piece the answer is written; else what its buffer holds, its rest's maximum and sum.
struct TopArgs {
    const void* x; size_t stride; int rows, n, k, pieces;
    float c; double T;
    float* values; long long* indices; float* rest;
    u64* part; float2* part_rest;                  // [rows][pieces][buffer_limit(k)], [rows][pieces]
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
            const u64 p = place(score_key(load_score(x, j)), j);
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
        const float v = load_score(x, j);
        if (place(score_key(v), j) < last) { if (v != v) rest.s = NAN; else rest.take(v, c); }
    }
    group_sync<W>();
}

// rest of the group: its threads' sums joined.  Every thread gets the pair.
template <int W> __device__ __forceinline__ void join_rest(Shared<W>& sh, int tid, const RestSum& r, float c, float& m, double& s) {
    const float own = W > 1 ? fmaxf(r.m, sh.far_m[tid]) : r.m;
    m = wave_reduce(own, OpFMax());
    if constexpr (W > 1) {
        if ((tid & 63) == 0) sh.rm[tid >> 6] = m;
        __syncthreads();
        for (int w = 0; w < W; ++w) m = fmaxf(m, sh.rm[w]);
    }
    s = (double)r.s * rebase(r.m, m, c);
    if constexpr (W > 1) s += sh.far_s[tid] * rebase(sh.far_m[tid], m, c);
    s = wave_reduce(s, OpSum());
    if constexpr (W > 1) {
        if ((tid & 63) == 0) sh.rs[tid >> 6] = s;
        __syncthreads();
        s = 0;
        for (int w = 0; w < W; ++w) s += sh.rs[w];
    }
}

// The k first of the buffer's n entries, in order, into the answer; the others into the rest.
template <int W> __device__ __forceinline__ void write_row(const TopArgs& a, size_t r, Shared<W>& sh, int tid, int n, RestSum& rest) {
    constexpr int G = W * 64;
    const int k = a.k;
    for (int i = tid; i < n; i += G) {
        const u64 p = sh.cand[i];
        int rank = 0;
#pragma unroll 8
        for (int o = 0; o < n; ++o) rank += sh.cand[o] > p ? 1 : 0;
        const float x = key_score((uint32_t)(p >> 32));
        if (rank < k) { a.values[r * k + rank] = x; a.indices[r * k + rank] = place_class(p); }
        else { if (x != x) rest.s = NAN; else rest.take(x, a.c); }
    }
}

// Waves a SIMD that the registers are cut for.  Measured at 4096 x 65536 bf16, k 64: 4 waves 223, 5 waves 207, 6 waves 233 us
// (spills); 2048 x 65536 float32: 4 waves 102, 5 waves 119 us (k 1); 200000 x 512 bf16, one wave a row, k 16: 247 / 228 / 220 us.
template <typename T, int W> constexpr int TOP_WAVES = W == 1 ? 6 : ET<T>::IS_BF16 ? 5 : 4;

template <typename T, int W>
__global__ __launch_bounds__(256, (TOP_WAVES<T, W>)) void top_scan_kernel(TopArgs a) {
    constexpr int VEC = ET<T>::VEC, G = W * 64, PER = 16, NB = PER / VEC, ROWS = W == 1 ? 4 : 1;
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

    if (tid == 0) sh.tau = 0;
    far_clear<W>(sh, tid);
    RestSum rest;
    int have = 0, turn = 0;                        // entries in the buffer
    i32x4 v[NB], nx[NB];
    auto load = [&](int b, i32x4* to) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int at = b * G * NB + i * G + tid;
            to[i] = load_vec(x, sp.vec_at(min(at, v1 - 1)));           // always: the last vector in the place of one beyond it
        }
    };
    if (v1 > 0) load(b0, nx);

    for (int b = b0; b < b1 || b == b0; ++b) {
        float f[PER];
        if ((b + 1) * G * NB > v1) {
#pragma unroll
            for (int i = 0; i < NB; ++i) if (b * G * NB + i * G + tid >= v1) nx[i] = neg_inf_vec<T>();
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) unpack16<T>(nx[i], f + i * VEC);
        if (b + 1 < b1) load(b + 1, nx);
        if (b == b0) {
            float top = f[0];
#pragma unroll
            for (int e = 1; e < PER; ++e) top = fmaxf(top, f[e]);
            // a bound that k scores of this batch reach, to 16 bits of the key: from 64 W maxima of threads, or 64 W NB of vectors
            const bool fine = W > 1 && k > 64;
            if (fine) {
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    float m = f[i * VEC];
#pragma unroll
                    for (int j = 1; j < VEC; ++j) m = fmaxf(m, f[i * VEC + j]);
                    sh.maxima[(i * G + tid) & (Shared<W>::EQ - 1)] = score_key(m);
                }
            } else sh.maxima[tid] = score_key(top);
            group_sync<W>();
            if (tid < 64) {
                const uint32_t t = bound_of_maxima<W == 1 ? 1 : W * NB>(sh.maxima, fine ? W * NB : W, k);
                // a bound at or below -inf: everything
                if (lane == 0) sh.lim = t <= KEY_NEG_INF ? NAN : score_before(t);
            }
            group_sync<W>();
        }
        // The first batch's bound is one that k scores reach.  A later batch's classes come after the buffer's: of those
        // only scores beyond the bound's are earlier in the order.  lim is NaN while there is no bound.
        const float lim = sh.lim;
        u64 mask[PER];                             // lanes whose score e may be among the first, in scalar registers
        u64 any = 0;
        int found = 0;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            mask[e] = __ballot(!(f[e] <= lim) && b * G * NB + (e / VEC) * G + tid < v1);
            any |= mask[e];
        }
        if (any) {
#pragma unroll
            for (int e = 0; e < PER; ++e) found += __popcll(mask[e]);
        }
        const int before = have;
        int slot = deal_slots<W>(sh, tid, have, turn, found);
        if (have <= Shared<W>::CAP) {
            if (found) {
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    if (mask[e]) {
                        if (mask[e] >> lane & 1) {
                            sh.cand[slot + lanes_below(mask[e])] = place(score_key(f[e]), sp.vec_at(b * G * NB + (e / VEC) * G + tid) + e % VEC);
                            f[e] = -INFINITY;
                        }
                        slot += __popcll(mask[e]);
                    }
                }
            }
            if (have > buffer_limit(k)) compact<T, W>(sh, tid, have, k, rest, c);
        } else {
            uint32_t pending = 0;
#pragma unroll
            for (int e = 0; e < PER; ++e) pending |= (uint32_t)(mask[e] >> lane & 1) << e;
            auto cls = [&](int e) { return sp.vec_at(b * G * NB + (e / VEC) * G + tid) + e % VEC; };
            have = before;
            const uint32_t kept = offer<T, W>(sh, tid, have, turn, k, pending, [&](int e) { return load_score(x, cls(e)); }, cls, rest, c);
#pragma unroll
            for (int e = 0; e < PER; ++e) if (kept >> e & 1) f[e] = -INFINITY;
        }
        // What is left is not beyond lim: with lim less than 60 octaves above the running maximum nothing can overflow, and
        // the batch's maximum need not be known.
        if (!((lim - rest.m) * c < 60.f)) {
            float top = f[0];
#pragma unroll
            for (int e = 1; e < PER; ++e) top = fmaxf(top, f[e]);
            rest.raise(top, c);
        }
        const float ref = rest.m == -INFINITY ? 0.f : rest.m;
#pragma unroll
        for (int e = 0; e < PER; ++e) rest.s += exp2_32((f[e] - ref) * c);
        if constexpr (W > 1) if (((b - b0) & (FLUSH - 1)) == FLUSH - 1) { far_add<W>(sh, tid, rest, c); rest.s = 0.f; }
    }
    // the row's ends, behind the last whole vector last in the order of classes; in front of the first they come first, so
    // those are held against the bound with their class
    for (int end = 0; end < 2; ++end) {
        const int some = end ? sp.edge - sp.head : sp.head, j = end ? n - some + tid : tid;
        if (!(end ? with_tail : with_head) || some == 0) continue;
        const float xe = tid < some ? load_score(x, j) : 0.f;
        const u64 tau = sh.tau;
        const bool maybe = tid < some && (tau ? place(score_key(xe), j) > tau : !(xe <= sh.lim));
        const uint32_t kept = offer<T, W>(sh, tid, have, turn, k, maybe ? 1u : 0u, [&](int) { return xe; }, [&](int) { return j; }, rest, c);
        if (tid < some && !kept) { if (xe != xe) rest.s = NAN; else rest.take(xe, c); }
    }
    if (have > G && a.pieces == 1) compact<T, W>(sh, tid, have, k, rest, c);
    else group_sync<W>();
    bool nan = rest.s != rest.s;
    if constexpr (W == 1) nan = __ballot(nan) != 0; else nan = __syncthreads_or(nan || sh.far_s[tid] != sh.far_s[tid]);
    if (nan) {
        const int lo = with_head ? 0 : sp.vec_at(b0 * G * NB), hi = with_tail ? n : sp.vec_at(v1);
        far_clear<W>(sh, tid);
        slow_row<T, W>(x, lo, hi, tid, k, sh, rest, c);
        have = min(k, hi - lo);
    }
    if (a.pieces == 1) write_row<W>(a, r, sh, tid, have, rest);
    float m; double s;
    join_rest<W>(sh, tid, rest, c, m, s);
    if (a.pieces == 1) {
        if (tid == 0) a.rest[r] = s != s ? NAN : m == -INFINITY ? -INFINITY : (float)((double)m / a.T + log(s));
    } else {
        const int limit = buffer_limit(k);
        for (int i = tid; i < limit; i += G) a.part[job * limit + i] = i < have ? sh.cand[i] : 0;
        if (tid == 0) a.part_rest[job] = make_float2(m, (float)s);
    }
}

// A row's pieces joined, as a first batch of at most MAX_MERGE places: a bound from the threads' maxima, the places that
// reach it into the buffer, the others into the rest.
constexpr int MAX_MERGE = 8192;
template <typename T>
__global__ __launch_bounds__(256) void top_merge_kernel(TopArgs a) {
    constexpr int R = MAX_MERGE / 256;
    __shared__ Shared<4> sh;
    const int tid = threadIdx.x, k = a.k, c = a.pieces * buffer_limit(k);
    const size_t r = blockIdx.x;
    const u64* part = a.part + r * c;
    uint32_t key[R], top[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < R; ++i) {
        key[i] = 0;
        if (256 * i < c && tid + 256 * i < c) key[i] = (uint32_t)(part[tid + 256 * i] >> 32);
        top[i & 3] = max(top[i & 3], key[i]);
    }
    far_clear<4>(sh, tid);
    RestSum rest;
    for (int i = tid; i < a.pieces; i += 256) {
        const float2 p = a.part_rest[r * a.pieces + i];
        rest.raise(p.x, a.c);
        rest.s += p.x == rest.m ? p.y : p.y * exp2_32((p.x - (rest.m == -INFINITY ? 0.f : rest.m)) * a.c);
    }
    const bool fine = k > 64;
    if (fine) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sh.maxima[256 * i + tid] = top[i];
    } else sh.maxima[tid] = max(max(top[0], top[1]), max(top[2], top[3]));
    __syncthreads();
    if (tid < 64) {
        const uint32_t t = bound_of_maxima<16>(sh.maxima, fine ? 16 : 4, k);
        if (tid == 0) sh.tau = (u64)t << 32;
    }
    __syncthreads();
    const uint32_t least = (uint32_t)(sh.tau >> 32);
    uint32_t pending = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) if (key[i] && key[i] >= least) pending |= 1u << i;
    int have = 0, turn = 0;
    const uint32_t kept = offer<T, 4>(sh, tid, have, turn, k, pending, [&](int e) { return key_score((uint32_t)(part[tid + 256 * e] >> 32)); },
                                      [&](int e) { return place_class(part[tid + 256 * e]); }, rest, a.c);
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (key[i] && !(kept >> i & 1)) { const float x = key_score(key[i]); if (x != x) rest.s = NAN; else rest.take(x, a.c); }
    if (have > 256) compact<T, 4>(sh, tid, have, k, rest, a.c);
    else __syncthreads();
    write_row<4>(a, r, sh, tid, have, rest);
    float m; double s;
    join_rest<4>(sh, tid, rest, a.c, m, s);
    if (tid == 0) a.rest[r] = s != s ? NAN : m == -INFINITY ? -INFINITY : (float)((double)m / a.T + log(s));
}

}  // namespace

// Pieces a row is split into.  512 rows fill the chip (two workgroups of four waves a compute unit) and are not split;
// fewer rows are cut into pieces of at least one batch (4096 scores) until 1024 workgroups run.  float32, k 64, us in 1 / 2 / 4 /
// 8 / 16 pieces: 32 x 65536 47 / 41 / 31 / 21 / 20, 128 x 65536 46 / 42 / 33 / 29 / 32, 256 x 65536 47 / 45 / 39 / 45 / 49,
// 512 x 65536 51 / 54 / 62 / 64 / 82, 2048 x 65536 123 / 164 / 201 / 205 / 297; 64 x 9000 18.0 / 19.6 / 18.5 in three, with k 5
// 11.3 / 17.6 / 16.8.
static int top_pieces(int rows, int ncls, int k) {
    if (rows >= 512 || ncls <= 512) return 1;
    const int batches = (ncls + 4095) / 4096;
    int p = (1024 + rows - 1) / rows;
    if (p > batches) p = batches;
    if (p * buffer_limit(k) > MAX_MERGE) p = MAX_MERGE / buffer_limit(k);
    return p;
}
static size_t top_workspace(int rows, int pieces, int k) { return pieces == 1 ? 0 : (size_t)rows * pieces * ((size_t)buffer_limit(k) * 8 + 8); }

extern "C" int stgcn_top_logits_workspace(int rows, int ncls, int k, size_t* bytes) {
    if (!bytes || rows < 1 || rows >= (1 << 24) || ncls < 1 || ncls > (1 << 20) || k < 1 || k > MAX_K || k > ncls) return STGCN_ERR_ARG;
    *bytes = top_workspace(rows, top_pieces(rows, ncls, k), k);
    return STGCN_OK;
}

extern "C" int stgcn_top_logits(int dtype, const void* logits, size_t row_stride, int rows, int ncls, int k, double temperature,
                                float* values, int64_t* indices, float* rest, void* workspace, size_t workspace_bytes, void* stream) {
    if (!logits || !values || !indices || !rest || rows < 1 || rows >= (1 << 24) || ncls < 1 || ncls > (1 << 20) || row_stride < (size_t)ncls || k < 1 || k > MAX_K
        || k > ncls || !temperature_ok(temperature) || (dtype != STGCN_F32 && dtype != STGCN_BF16)) return STGCN_ERR_ARG;
    const int pieces = top_pieces(rows, ncls, k);
    if (pieces > 1 && (!workspace || workspace_bytes < top_workspace(rows, pieces, k))) return STGCN_ERR_WORKSPACE;
    TopArgs a = {logits, row_stride, rows, ncls, k, pieces, (float)(LOG2E / temperature), temperature, values, (long long*)indices, rest,
                 (u64*)workspace, (float2*)((char*)workspace + (pieces > 1 ? (size_t)rows * pieces * buffer_limit(k) * 8 : 0))};
    const hipStream_t s = (hipStream_t)stream;
    const unsigned grid = ncls <= 512 ? (unsigned)((rows + 3) / 4) : (unsigned)rows * pieces;
    if (dtype == STGCN_BF16) {
        if (ncls <= 512) top_scan_kernel<bf16, 1><<<grid, 256, 0, s>>>(a); else top_scan_kernel<bf16, 4><<<grid, 256, 0, s>>>(a);
        if (pieces > 1) top_merge_kernel<bf16><<<rows, 256, 0, s>>>(a);
    } else {
        if (ncls <= 512) top_scan_kernel<float, 1><<<grid, 256, 0, s>>>(a); else top_scan_kernel<float, 4><<<grid, 256, 0, s>>>(a);
        if (pieces > 1) top_merge_kernel<float><<<rows, 256, 0, s>>>(a);
    }
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}
