// A label per row drawn from class scores with given random numbers.
//
// With w_j = e^{(x_j - max x) / T} and the classes in the order (score descending, class ascending):
//   keep the first top_k (0: all); of these the shortest prefix whose sum reaches top_p times the sum of all of these;
//   of these those with w_j >= min_p (the first class is always kept);
//   answer the first kept class j, by class number, with  sum_{i <= j, kept} w_i > u * sum of the kept w.
// All three cuts keep a prefix of that order, so the kept set is a pair (score xt, class ti): every class with a larger
// score, and of the classes with that score those up to ti.  Weights and sums are held in 64 bits: the answer is a whole
// number, and a sum in 32 bits would move it wherever u falls within 1e-7 of a border between two classes.
//
// One workgroup a row.  Every look at the row is a pass over it; after the first one it comes from the caches (a row in
// registers was tried: fully unrolled passes with 64-bit weights spill).  What the cuts need of it:
//   top_k up to a few hundred: k of the threads' maxima reach a bound that about k to 2k scores reach; those go to a list
//     in LDS, where everything else happens, and no weight of any other class is computed;
//   larger top_k, and top_p: the scores (or their weights) counted by 128 bins of the score; the bin in which the count
//     (the sum) crosses gives a short list, in which the border is bisected.  Bins and list hold weights as 64-bit integers
//     in units of 2^-s (s = 42 to 50 by the class count): their sums are the same in any order.  A border that falls within
//     such a unit of a class moves that class alone, by a share of 2^-s of the first class's weight;
//   the answer: sums of the kept weights by cells (64 consecutive vectors: one wave's step), the cell in which u falls,
//     then the lane, then the class.
#include "scores.h"

namespace {

constexpr double LOG2E = 1.4426950408889634074;
constexpr int BINS = 128;
typedef unsigned long long u64;

struct SampleArgs {
    const void* x; size_t stride; const float* u;
    const float* tp; const int* kp; const float* pp; const float* qp;      // per row, or null: the scalars
    float t; int k; float p, q;
    long long* labels; float* logp; int n;
};

__device__ __forceinline__ u64 place(uint32_t key, int j) { return ((u64)key << 32) | (uint32_t)~j; }
__device__ __forceinline__ int place_class(u64 p) { return (int)~(uint32_t)p; }
__device__ __forceinline__ float place_score(u64 p) { return key_score((uint32_t)(p >> 32)); }

// Weights relative to the row's maximum.  With a maximum of +inf its classes weigh 1, all others nothing.
struct Weight {
    double xmax, c, unit; bool inf;                // unit: 2^(52 - s); the low 52 bits of w + unit are w in units of 2^-s
    __device__ __forceinline__ u64 fixed(double w) const { return (u64)__double_as_longlong(w + unit) & ((1ull << 52) - 1); }
    __device__ __forceinline__ double operator()(float x) const {
        if (inf) return x == INFINITY ? 1.0 : 0.0;
        return exp2_64(((double)x - xmax) * c);
    }
    template <int N> __device__ __forceinline__ void many(const float* x, double* w) const {
        if (inf) {
#pragma unroll
            for (int e = 0; e < N; ++e) w[e] = x[e] == INFINITY ? 1.0 : 0.0;
            return;
        }
        double y[N];
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = ((double)x[e] - xmax) * c;
        exp2_64<N>(y, w);
    }
};

// The kept set: x > xt, or x == xt and class <= ti.
struct Cut {
    float xt; int ti;
    __device__ __forceinline__ bool operator()(float x, int j) const { return x > xt || (x == xt && j <= ti); }
};

template <int W, int CELLS> struct Shared {
    static constexpr int CAP = W * 256;            // four places a thread
    static constexpr int COPIES = 32;              // of the bins, one a lane of a half wave, each in banks of its own: a
    union {                                        // wave's adds never meet, whatever the scores
        u64 bins[BINS][COPIES];
        struct { u64 list[CAP]; double mass[CAP]; } l;
    };
    union { double sum[CELLS]; int count[CELLS]; } cell;
    u64 total[BINS];
    double all; u64 redu[W]; int redi[W]; uint32_t red2[2][W];
    int pick; double before; Cut cut;
};

// One row as its workgroup of W waves sees it: steps of one vector a thread.
// Cells in the order of the classes: the row's front end, then vector cells (step i, wave w), then its back end.
template <typename T, int W> struct Row {
    static constexpr int VEC = ET<T>::VEC, G = W * 64;
    const T* x;
    RowSpan<T> sp;
    int n, tid, lane, wave, steps;
    float xe;                                      // of the threads below sp.edge

    __device__ __forceinline__ Row(const T* x_, int n_) : x(x_), sp(x_, n_), n(n_), tid(threadIdx.x), lane(threadIdx.x & 63), wave(threadIdx.x >> 6) {
        steps = (sp.nvec + G - 1) / G;
        xe = tid < sp.edge ? load_elem(x, sp.edge_at(tid)) : -INFINITY;
    }
    __device__ __forceinline__ i32x4 load(int i) const { return i * G + tid < sp.nvec ? load_vec(x, sp.vec_at(i * G + tid)) : neg_inf_vec<T>(); }
    __device__ __forceinline__ bool valid(int i) const { return i * G + tid < sp.nvec; }
    __device__ __forceinline__ int cls(int i, int e) const { return sp.vec_at(i * G + tid) + e; }
    __device__ __forceinline__ int cells() const { return steps * W + 2; }
    __device__ __forceinline__ int cell(int i) const { return 1 + i * W + wave; }
    // f(i, scores of vector i); scores beyond the row are -inf.  Three steps' loads are under way at a time.
    template <typename F> __device__ __forceinline__ void each(F f) const {
        i32x4 v0 = load(0), v1 = load(1), v2 = load(2);
#pragma unroll 1
        for (int i = 0; i < steps; ++i) {
            float s[VEC];
            unpack16<T>(v0, s);
            v0 = v1; v1 = v2; v2 = load(i + 3);
            f(i, s);
        }
    }
    // f(scores of vector i), by the wave that has that cell
    template <typename F> __device__ __forceinline__ void at_cell(int c, F f) const {
        const int i = (c - 1) / W;
        if (c < 1 || c > steps * W || (c - 1) % W != wave) return;
        float s[VEC];
        unpack16<T>(load(i), s);
        f(i, s);
    }
};

// Largest v in [lo, hi] with enough(v), which holds at lo.
template <typename F> __device__ __forceinline__ uint32_t last_enough(uint32_t lo, uint32_t hi, F enough) {
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if (enough(mid)) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// How many of `ties` equal weights `one` the sum needs to get from `over` to target: at least one, at most all.
__device__ __forceinline__ int ties_needed(u64 over, u64 one, u64 target, int ties) {
    if (one == 0 || over + one >= target) return one == 0 ? ties : 1;
    const u64 m = (target - over + one - 1) / one;
    return m < (u64)ties ? (int)m : ties;
}

// Places in LDS, four a thread of a workgroup of W waves or, for lists of at most 256, of its first wave alone (V = 1: no
// barriers).
template <typename T, int V, typename S> struct List {
    static constexpr int G = V * 64;
    static constexpr int SHIFT = ET<T>::IS_BF16 ? 16 : 0;                  // bits of a key that carry nothing
    S& sh;
    int tid, lane, wave, n;                        // n: classes of the row
    u64 lp[4]; double lw[4];
    __device__ __forceinline__ List(S& s, int c, int n_, const Weight& weight) : sh(s), tid(threadIdx.x), lane(threadIdx.x & 63), wave(threadIdx.x >> 6), n(n_) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { lp[i] = tid + G * i < c ? sh.l.list[tid + G * i] : 0; lw[i] = lp[i] ? weight(place_score(lp[i])) : 0.0; }
    }
    template <typename P> __device__ __forceinline__ int count(P pred) {
        int m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m += __popcll(__ballot(lp[i] && pred(lp[i])));
        if constexpr (V == 1) return m;
        __syncthreads();
        if (lane == 0) sh.redi[wave] = m;
        __syncthreads();
        m = 0;
#pragma unroll
        for (int w = 0; w < V; ++w) m += sh.redi[w];
        return m;
    }
    // weights of the entries that pass, in integer units
    template <typename P> __device__ __forceinline__ u64 mass(const Weight& weight, P pred) {
        u64 m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) if (lp[i] && pred(lp[i])) m += weight.fixed(lw[i]);
        m = wave_sum(m);
        if constexpr (V == 1) return m;
        __syncthreads();
        if (lane == 0) sh.redu[wave] = m;
        __syncthreads();
        m = 0;
#pragma unroll
        for (int w = 0; w < V; ++w) m += sh.redu[w];
        return m;
    }
    __device__ __forceinline__ void range(uint32_t& lo, uint32_t& hi) {
        uint32_t l = 0, h = 0;                     // ~ of the smallest key, the largest
#pragma unroll
        for (int i = 0; i < 4; ++i) if (lp[i]) { l = max(l, ~key(lp[i])); h = max(h, key(lp[i])); }
        lo = ~block_reduce<V>(l, OpMax(), sh.red2[0]);
        hi = block_reduce<V>(h, OpMax(), sh.red2[1]);
    }
    static __device__ __forceinline__ uint32_t key(u64 e) { return (uint32_t)(e >> (32 + SHIFT)); }
    static __device__ __forceinline__ float score(uint32_t s) { return key_score(ET<T>::IS_BF16 ? s << 16 | ((s & 0x8000u) ? 0u : 0xFFFFu) : s); }
    // the m-th by class of the entries with key v
    __device__ __forceinline__ int tie(uint32_t v, int m) {
        return (int)~last_enough(~(uint32_t)(n - 1), ~0u, [&](uint32_t mid) { return count([&](u64 e) { return key(e) == v && (uint32_t)e >= mid; }) >= m; });
    }
    // the first k entries
    __device__ __forceinline__ Cut cut_count(int k) {
        uint32_t lo, hi;
        range(lo, hi);
        const uint32_t v = last_enough(lo, hi, [&](uint32_t mid) { return count([&](u64 e) { return key(e) >= mid; }) >= k; });
        const int above = count([&](u64 e) { return key(e) > v; }), ties = count([&](u64 e) { return key(e) == v; });
        return {score(v), above + ties > k ? tie(v, k - above) : n};
    }
    // the shortest prefix that, after `above`, reaches the target; `was`: what cut the entries so far
    __device__ __forceinline__ Cut cut_mass(u64 above, u64 target, const Weight& weight, const Cut& was) {
        uint32_t lo, hi;
        range(lo, hi);
        const uint32_t v = last_enough(lo, hi, [&](uint32_t mid) { return above + mass(weight, [&](u64 e) { return key(e) >= mid; }) >= target; });
        const u64 over = above + mass(weight, [&](u64 e) { return key(e) > v; });
        const int ties = count([&](u64 e) { return key(e) == v; });
        const float x = score(v);
        const int m = ties_needed(over, weight.fixed(weight(x)), target, ties);
        return {x, m < ties ? tie(v, m) : x == was.xt ? was.ti : n};
    }
    __device__ __forceinline__ u64 all(const Weight& weight) { return mass(weight, [](u64) { return true; }); }
    __device__ __forceinline__ void keep(const Cut& cut) {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (lp[i] && !cut(place_score(lp[i]), place_class(lp[i]))) { lp[i] = 0; lw[i] = 0; }
    }
    // The answer, from entries that are all there is: (class, log of its share) by one thread.
    template <typename A> __device__ __forceinline__ void draw(float u, double least, A answer) {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (lw[i] == 0 || lw[i] < least) lp[i] = 0;
        int c = 0;                                 // packed: places and weights
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u64 b = __ballot(lp[i] != 0);
            int at = c;
            if constexpr (V == 1) c += __popcll(b);
            else {
                __syncthreads();
                if (lane == 0) sh.redi[wave] = __popcll(b);
                __syncthreads();
                for (int w = 0; w < V; ++w) { if (w < wave) at += sh.redi[w]; c += sh.redi[w]; }
            }
            if (lp[i]) { sh.l.list[at + lanes_below(b)] = lp[i]; sh.l.mass[at + lanes_below(b)] = lw[i]; }
        }
        if constexpr (V == 1) { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier(); } else __syncthreads();
        double all = 0, front[4] = {0, 0, 0, 0};   // the mass of lower classes
        for (int o = 0; o < c; ++o) {
            const u64 e = sh.l.list[o];
            const double w = sh.l.mass[o];
            all += w;
#pragma unroll
            for (int i = 0; i < 4; ++i) if ((uint32_t)e > (uint32_t)lp[i]) front[i] += w;
        }
        const double target = (double)u * all;
        // the first class whose sum exceeds the target; the last one if rounding leaves none.  Lower class = larger ~class.
        u64 best = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lp[i]) best = max(best, front[i] + lw[i] > target ? (1ull << 32) | (uint32_t)lp[i] : (u64)(uint32_t)~(uint32_t)lp[i] + 1);
        best = block_reduce<V>(best, OpMax(), sh.redu);
        const uint32_t who = best >> 32 ? (uint32_t)best : ~(uint32_t)(best - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) if (lp[i] && (uint32_t)lp[i] == who) answer(place_class(lp[i]), (float)log(lw[i] / all));
    }
};

template <typename T, int W, int CELLS>
__global__ __launch_bounds__(W * 64) void sample_kernel(SampleArgs a) {
    typedef Row<T, W> R;
    typedef Shared<W, CELLS> S;
    constexpr int VEC = R::VEC, G = R::G, CAP = S::CAP;
    __shared__ S sh;
    const size_t r = blockIdx.x;
    const R row((const T*)((const char*)a.x + r * a.stride * ET<T>::ES), a.n);
    const int tid = row.tid, lane = row.lane, wave = row.wave, n = a.n;
    const float u = a.u[r], t = a.tp ? a.tp[r] : a.t, p = a.pp ? a.pp[r] : a.p, q = a.qp ? a.qp[r] : a.q;
    int k = a.kp ? a.kp[r] : a.k;
    auto answer = [&](int label, float lp) { a.labels[r] = label; a.logp[r] = lp; };       // by one thread

    // the row's maximum, its smallest finite score, and whether a NaN is there
    float mine = row.xe, low = row.xe > -INFINITY ? row.xe : INFINITY;
    bool nan = row.xe != row.xe;
    row.each([&](int i, const float* s) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) { mine = fmaxf(mine, s[e]); nan |= s[e] != s[e]; low = fminf(low, s[e] > -INFINITY ? s[e] : INFINITY); }
    });
    const uint32_t top = block_reduce<W>(nan ? KEY_NAN : score_key(mine), OpMax(), sh.red2[0]);
    if (top == KEY_NAN || !(t >= 0.f) || !(t < INFINITY) || k < 0 || !(p > 0.f) || !(p <= 1.f) || !(q >= 0.f) || !(q <= 1.f) || !(u >= 0.f) || !(u < 1.f)) {
        if (tid == 0) answer(-1, NAN);
        return;
    }
    if (top == KEY_NEG_INF) { if (tid == 0) answer(-1, -INFINITY); return; }
    const float xmax = key_score(top);
    const int s = min(50, 30 + __clz(n));          // n sums of at most 2^s stay below 2^63
    const Weight weight = {(double)xmax, t > 0.f ? LOG2E / (double)t : 0.0, (double)(1ull << (52 - s)), xmax == INFINITY};
    if (t == 0.f || k == 1) {
        int at = n;
        row.each([&](int i, const float* s) {
#pragma unroll
            for (int e = VEC - 1; e >= 0; --e) if (s[e] == xmax) at = min(at, row.cls(i, e));
        });
        if (tid < row.sp.edge && row.xe == xmax) at = min(at, row.sp.edge_at(tid));
        at = (int)~block_reduce<W>(~(uint32_t)at, OpMax(), sh.red2[1]);
        if (tid == 0) answer(at, 0.f);
        return;
    }
    if (k == 0 || k > n) k = n;

    Cut cut = {-INFINITY, n};
    // Scores of a vector that are not kept become -inf, which weighs nothing.  False: none of the wave's is kept.
    auto only_kept = [&](int i, const float* s, float* x, float lowest) {
        const float lo = fmaxf(cut.xt, lowest);
        bool some = false;
#pragma unroll
        for (int e = 0; e < VEC; ++e) { x[e] = s[e] >= lo ? s[e] : -INFINITY; some |= s[e] >= lo; }
        if (!__ballot(some)) return false;
        if (cut.ti < n) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) if (s[e] == cut.xt && row.cls(i, e) > cut.ti) x[e] = -INFINITY;
        }
        return true;
    };
    auto mass_target = [&](u64 all) { return (u64)ceil((double)p * (double)all); };
    auto count_waves = [&](int m) {                // sum over the waves of a number that is the same in a wave's lanes
        __syncthreads();
        if (lane == 0) sh.redi[wave] = m;
        __syncthreads();
        int s = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) s += sh.redi[w];
        return s;
    };
    // scores that pass, counted
    auto count = [&](auto pred) {
        int m = 0;
        row.each([&](int i, const float* s) {
            const bool ok = row.valid(i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) m += __popcll(__ballot(ok && pred(s[e], row.cls(i, e))));
        });
        if (wave == 0) m += __popcll(__ballot(tid < row.sp.edge && pred(row.xe, row.sp.edge_at(tid))));
        return count_waves(m);
    };
    // weights of the scores that pass, in integer units
    auto mass = [&](auto pred) {
        u64 m = 0;
        row.each([&](int i, const float* s) {
            const bool ok = row.valid(i);
            float x[VEC];
            bool some = false;
#pragma unroll
            for (int e = 0; e < VEC; ++e) { const bool in = ok && pred(s[e], row.cls(i, e)); x[e] = in ? s[e] : -INFINITY; some |= in; }
            if (!__ballot(some)) return;
            double w[VEC];
            weight.template many<VEC>(x, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) m += weight.fixed(w[e]);
        });
        if (tid < row.sp.edge && pred(row.xe, row.sp.edge_at(tid))) m += weight.fixed(weight(row.xe));
        return block_reduce<W>(m, OpSum(), sh.redu);
    };
    // counts by cells of the scores that pass, as prefix sums: cell.count[c] = how many lie in front of cell c.  Returns all.
    auto count_cells = [&](auto pred) {
        __syncthreads();
        const int cells = row.cells();
        row.each([&](int i, const float* s) {
            const bool ok = row.valid(i);
            int m = 0;
#pragma unroll
            for (int e = 0; e < VEC; ++e) m += __popcll(__ballot(ok && pred(s[e], row.cls(i, e))));
            if (lane == 0) sh.cell.count[row.cell(i)] = m;
        });
        if (wave == 0) {
            const u64 b = __ballot(tid < row.sp.edge && pred(row.xe, row.sp.edge_at(tid))), front = (1ull << row.sp.head) - 1;
            if (lane == 0) { sh.cell.count[0] = __popcll(b & front); sh.cell.count[cells - 1] = __popcll(b & ~front); }
        }
        __syncthreads();
        if (wave == 0) {
            int run = 0;
            for (int c = 0; c < cells; c += 64) {
                const int m = c + lane < cells ? sh.cell.count[c + lane] : 0;
                int s = m;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(s, d); if (lane >= d) s += o; }
                if (c + lane < cells) sh.cell.count[c + lane] = run + s - m;
                run += __shfl(s, 63);
            }
            if (lane == 0) sh.pick = run;
        }
        __syncthreads();
        return sh.pick;
    };
    // The scores that pass, as places in the list (in no particular order: everything that is made of it is a set, or a sum
    // of integers).  Returns how many there are; more than CAP are not all in it.
    auto collect = [&](auto pred) {
        __syncthreads();
        if (tid == 0) sh.pick = 0;
        __syncthreads();
        auto append = [&](bool in, float x, int j) {
            const u64 b = __ballot(in);
            if (b) {
                int at = 0;
                if (lane == 0) at = atomicAdd(&sh.pick, __popcll(b));
                at = __builtin_amdgcn_readfirstlane(at) + lanes_below(b);
                if (in && at < CAP) sh.l.list[at] = place(score_key(x), j);
            }
        };
        row.each([&](int i, const float* s) {
            const bool ok = row.valid(i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) append(ok && pred(s[e], row.cls(i, e)), s[e], row.cls(i, e));
        });
        if (wave == 0) append(tid < row.sp.edge && pred(row.xe, row.sp.edge_at(tid)), row.xe, row.sp.edge_at(tid));
        __syncthreads();
        const int c = sh.pick;
        __syncthreads();
        return c;
    };
    // The class of the m-th one, by class, of the scores equal to x.
    auto nth = [&](float x, int m) {
        auto is = [&](float s, int) { return s == x; };
        count_cells(is);
        if (wave == 0) {                           // the last cell with fewer than m in front of it
            int c = 0;
            for (int b = 0; b < row.cells(); b += 64) {
                const bool in = b + lane < row.cells() && sh.cell.count[b + lane] < m;
                c += __popcll(__ballot(in));
            }
            if (lane == 0) sh.pick = c - 1;
        }
        __syncthreads();
        const int c = sh.pick, cells = row.cells();
        const int left = m - sh.cell.count[c];     // the left-th one of that cell
        row.at_cell(c, [&](int i, const float* s) {
            int own = 0;
            const bool ok = row.valid(i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) own += ok && s[e] == x ? 1 : 0;
            int s0 = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(s0, d); if (lane >= d) s0 += o; }
            if (s0 - own < left && left <= s0) {
                int rank = s0 - own;
#pragma unroll
                for (int e = 0; e < VEC; ++e) if (s[e] == x && ++rank == left) sh.redi[0] = row.cls(i, e);
            }
        });
        if (wave == 0 && (c == 0 || c == cells - 1)) {
            const u64 b = __ballot(tid < row.sp.edge && row.xe == x), front = (1ull << row.sp.head) - 1, here = c == 0 ? b & front : b & ~front;
            if ((here >> lane & 1) && lanes_below(here) == left - 1) sh.redi[0] = row.sp.edge_at(tid);
        }
        __syncthreads();
        const int j = sh.redi[0];
        __syncthreads();
        return j;
    };
    constexpr int SHIFT = ET<T>::IS_BF16 ? 16 : 0; // bits of a key that carry nothing
    auto wide_key = [](uint32_t s) { return ET<T>::IS_BF16 ? s << 16 | ((s & 0x8000u) ? 0u : 0xFFFFu) : s; };

    // min_p: a weight is only computed where a 32-bit estimate of the border, with room, says that it may pass
    const double least = q > 0.f ? (double)q : 0.0;
    const float xq = q > 0.f && !weight.inf ? (float)((double)xmax + (log2((double)q) - 1e-3) / weight.c) : -INFINITY;
    const float xlow = xq - fabsf(xq) * 1e-6f;

    // ---- borders ----------------------------------------------------------------------------------------------------
    // The kept scores (`cut`) by bins: one each, or their weights.
    float scale = 0.f;                             // quarter octaves of the weight, or finer where the row is narrower
    auto bin = [&](float x) { return (int)fminf((xmax - x) * scale, (float)(BINS - 1)); };
    auto in_bin = [&](float x, int b) { const float f = (xmax - x) * scale; return b < BINS - 1 ? f >= (float)b && f < (float)(b + 1) : !(f < (float)b); };
    auto fill_bins = [&](bool weigh) {
        const float smallest = key_score(~block_reduce<W>(~score_key(low), OpMax(), sh.red2[0]));
        scale = (float)fmin(4.0 * weight.c, 1e30);
        if ((xmax - smallest) * scale < (float)(BINS - 1) && xmax > smallest) scale = (float)(BINS - 1) / (xmax - smallest);
        __syncthreads();
        for (int i = tid; i < S::COPIES * BINS; i += G) (&sh.bins[0][0])[i] = 0;
        __syncthreads();
        auto drop = [&](float x, u64 v) { atomicAdd(&sh.bins[bin(x)][lane & 31], v); };
        row.each([&](int i, const float* s) {
            float x[VEC];
            if (!only_kept(i, s, x, -INFINITY)) return;
            if (weigh) {
                double w[VEC];
                weight.template many<VEC>(x, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) drop(s[e], weight.fixed(w[e]));
            } else {
                const u64 one = row.valid(i) ? 1 : 0;  // top_k comes first: every score counts
#pragma unroll
                for (int e = 0; e < VEC; ++e) drop(s[e], one);
            }
        });
        if (tid < row.sp.edge && cut(row.xe, row.sp.edge_at(tid))) drop(row.xe, weigh ? weight.fixed(weight(row.xe)) : 1);
        __syncthreads();
        for (int b = tid; b < BINS; b += G) {
            u64 s = 0;
            for (int i = 0; i < S::COPIES; ++i) s += sh.bins[b][(i + tid) & (S::COPIES - 1)];
            sh.total[b] = s;
        }
        __syncthreads();
    };
    // Sum of the bins; the first bin at which the running sum reaches target (by every wave: two bins a lane).
    auto bin_sum = [&]() { return wave_sum(sh.total[2 * lane] + sh.total[2 * lane + 1]); };
    auto bin_reach = [&](u64 target, u64& above) {
        const u64 a0 = sh.total[2 * lane], a1 = sh.total[2 * lane + 1];
        u64 s = a0 + a1;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const u64 o = __shfl_up(s, d); if (lane >= d) s += o; }
        const u64 hit = __ballot(s >= target);
        const int l = hit ? __ffsll(hit) - 1 : 63;
        const u64 f = __shfl(s, l) - __shfl(a0 + a1, l), m0 = __shfl(a0, l);   // in front of the pair, its first
        const bool second = f + m0 < target;
        above = second ? f + m0 : f;
        return 2 * l + (second ? 1 : 0);
    };
    // list(c): work on a list of c places by the first wave alone if they are few; its cut to all
    auto with_list = [&](int c, auto work) {
        if (c <= 256) {
            if (wave == 0) { List<T, 1, S> list(sh, c, n, weight); const Cut to = work(list); if (lane == 0) sh.cut = to; }
            __syncthreads();
            cut = sh.cut;
        } else { List<T, W, S> list(sh, c, n, weight); cut = work(list); }
    };
    // What equal scores x leave of it: all, or the first `need` by class.
    auto cut_ties = [&](float x, int need, int ties) { cut = {x, need < ties ? nth(x, need) : x == cut.xt ? cut.ti : n}; };

    // ---- top_k ------------------------------------------------------------------------------------------------------
    if (k < n) {
        if (k <= G / 2) {                          // k of the threads' maxima reach a bound
            const uint32_t key = score_key(mine) >> SHIFT;
            const uint32_t v = last_enough(0, top >> SHIFT, [&](uint32_t mid) { return count_waves(__popcll(__ballot(key >= mid))) >= k; });
            const float bound = wide_key(v) > KEY_NEG_INF ? key_score(wide_key(v)) : NAN;
            const int c = collect([&](float s, int) { return s >= bound; });
            if (c >= k && c <= CAP) {
                // the list holds everything: top_k, top_p and the answer from it
                auto rest = [&](auto list) {
                    cut = list.cut_count(k);
                    list.keep(cut);
                    if (p < 1.f) { cut = list.cut_mass(0, mass_target(list.all(weight)), weight, cut); list.keep(cut); }
                    list.draw(u, least, answer);
                };
                if (c <= 256) { if (wave == 0) rest(List<T, 1, S>(sh, c, n, weight)); }
                else rest(List<T, W, S>(sh, c, n, weight));
                return;
            }
        }
        fill_bins(false);
        u64 above;
        const int b = bin_reach((u64)k, above);
        const int c = collect([&](float x, int) { return in_bin(x, b); }), need = k - (int)above;
        if (c <= CAP) with_list(c, [&](auto& list) { return list.cut_count(need); });
        else {                                     // many equal or nearly equal scores: bisection over the row
            const uint32_t v = last_enough(0, top >> SHIFT, [&](uint32_t mid) {
                const float s = key_score(wide_key(mid));
                return wide_key(mid) <= KEY_NEG_INF || count([&](float x, int) { return x >= s; }) >= k; });
            if (wide_key(v) > KEY_NEG_INF) {       // else only scores of -inf, which weigh nothing, are cut
                const float x = key_score(wide_key(v));
                const int over = count([&](float s, int) { return s > x; }), ties = count([&](float s, int) { return s == x; });
                cut_ties(x, k - over, ties);
            }
        }
    }
    // ---- top_p ------------------------------------------------------------------------------------------------------
    if (p < 1.f) {
        if (n <= CAP) {                            // a row that fits in the list
            const int c = collect(cut);
            with_list(c, [&](auto& list) { return list.cut_mass(0, mass_target(list.all(weight)), weight, cut); });
        } else {
            fill_bins(true);
            const u64 target = mass_target(bin_sum());
            u64 above;
            const int b = bin_reach(target, above);
            const int c = collect([&](float x, int j) { return in_bin(x, b) && cut(x, j); });
            if (c <= CAP) with_list(c, [&](auto& list) { return list.cut_mass(above, target, weight, cut); });
            else {
                const float x = key_score(wide_key(last_enough(0, top >> SHIFT, [&](uint32_t mid) {
                    const float s = key_score(wide_key(mid));
                    return wide_key(mid) <= KEY_NEG_INF || mass([&](float x, int j) { return x >= s && cut(x, j); }) >= target; })));
                const u64 over = mass([&](float s, int j) { return s > x && cut(s, j); });
                const int ties = count([&](float s, int j) { return s == x && cut(s, j); });
                cut_ties(x, ties_needed(over, weight.fixed(weight(x)), target, ties), ties);
            }
        }
    }
    // ---- the answer -------------------------------------------------------------------------------------------------
    auto share = [&](float x, int j) {             // the weight of a class that is kept, else 0
        double w = 0;
        if (x >= xlow && cut(x, j)) { w = weight(x); if (w < least) w = 0; }
        return w;
    };
    __syncthreads();
    row.each([&](int i, const float* s) {
        double m = 0;
        float x[VEC];
        if (only_kept(i, s, x, xlow)) {
            double w[VEC];
            weight.template many<VEC>(x, w);
            if (least > 0) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) w[e] = w[e] >= least ? w[e] : 0.0;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) m += w[e];
            m = wave_sum(m);
        }
        if (lane == 0) sh.cell.sum[row.cell(i)] = m;
    });
    const int cells = row.cells();
    if (wave == 0) {
        const double w = tid < row.sp.edge ? share(row.xe, row.sp.edge_at(tid)) : 0.0;
        const double f = wave_sum(tid < row.sp.head ? w : 0.0), b = wave_sum(tid < row.sp.head ? 0.0 : w);
        if (lane == 0) { sh.cell.sum[0] = f; sh.cell.sum[cells - 1] = b; }
    }
    __syncthreads();
    double all = 0;
    if (wave == 0) {
        for (int c = 0; c < cells; c += 64) all += wave_sum(c + lane < cells ? sh.cell.sum[c + lane] : 0.0);
        const double target = (double)u * all;
        // the first cell whose running sum exceeds the target, or the last one that holds anything
        double run = 0, found_before = 0;
        int found = -1, last = 0; double last_before = 0;
        for (int c = 0; c < cells; c += 64) {
            const double m = c + lane < cells ? sh.cell.sum[c + lane] : 0.0;
            double s = m;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) { const double o = __shfl_up(s, d); if (lane >= d) s += o; }
            const u64 hit = __ballot(m > 0 && run + s > target), some = __ballot(m > 0);
            if (some) { const int l = 63 - __clzll(some); last = c + l; last_before = run + __shfl(s - m, l); }
            if (hit) { const int l = __ffsll(hit) - 1; found = c + l; found_before = run + __shfl(s - m, l); break; }
            run += __shfl(s, 63);
        }
        if (lane == 0) { sh.pick = found >= 0 ? found : last; sh.before = found >= 0 ? found_before : last_before; sh.all = all; }
    }
    __syncthreads();
    const int c = sh.pick;
    const double before = sh.before;
    all = sh.all;
    const double target = (double)u * all;
    auto finish = [&](const double* w, const int* cl, int m) {             // one wave: m weights a lane, classes ascending over lanes
        double own = 0;
        for (int e = 0; e < m; ++e) own += w[e];
        double s = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const double o = __shfl_up(s, d); if (lane >= d) s += o; }
        const double front = before + (s - own);
        int hit = -1; double hw = 0, run = front;
        int lastc = -1; double lastw = 0;
        for (int e = 0; e < m; ++e) {
            run += w[e];
            if (w[e] > 0) { lastc = cl[e]; lastw = w[e]; if (hit < 0 && run > target) { hit = cl[e]; hw = w[e]; } }
        }
        const u64 b = __ballot(hit >= 0), l = __ballot(lastc >= 0);
        const int who = b ? __ffsll(b) - 1 : 63 - __clzll(l);
        if (lane == who) answer(b ? hit : lastc, (float)log((b ? hw : lastw) / all));
    };
    row.at_cell(c, [&](int i, const float* s) {
        double w[VEC]; int cl[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) { cl[e] = row.cls(i, e); w[e] = row.valid(i) ? share(s[e], cl[e]) : 0.0; }
        finish(w, cl, VEC);
    });
    if (wave == 0 && (c == 0 || c == cells - 1)) {
        const bool here = tid < row.sp.edge && (tid < row.sp.head) == (c == 0);
        const int j = here ? row.sp.edge_at(tid) : 0;
        const double w = here ? share(row.xe, j) : 0.0;
        finish(&w, &j, 1);
    }
}

template <typename T> void launch(const SampleArgs& a, int rows, hipStream_t s) {
    constexpr int VEC = ET<T>::VEC;
    const int nv = a.n / VEC;
    if (a.n <= 256) sample_kernel<T, 1, 4><<<rows, 64, 0, s>>>(a);
    else if (nv <= 2048) sample_kernel<T, 4, 34><<<rows, 256, 0, s>>>(a);
    else sample_kernel<T, 16, (1 << 20) / VEC / 64 + 18><<<rows, 1024, 0, s>>>(a);
}

}  // namespace

extern "C" int stgcn_sample_labels(int dtype, const void* logits, size_t row_stride, const float* u, const float* temperatures, float temperature,
                                   const int* top_ks, int top_k, const float* top_ps, float top_p, const float* min_ps, float min_p,
                                   int64_t* labels, float* logp, int rows, int ncls, void* stream) {
    if (!logits || !u || !labels || !logp || rows < 1 || ncls < 1 || ncls > (1 << 20) || row_stride < (size_t)ncls) return STGCN_ERR_ARG;
    SampleArgs a = {logits, row_stride, u, temperatures, top_ks, top_ps, min_ps, temperature, top_k, top_p, min_p, (long long*)labels, logp, ncls};
    if (dtype == STGCN_BF16) launch<bf16>(a, rows, (hipStream_t)stream);
    else if (dtype == STGCN_F32) launch<float>(a, rows, (hipStream_t)stream);
    else return STGCN_ERR_ARG;
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}
