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
//   larger top_k, and top_p: the scores (or their weights) counted by bins of the score; the bin in which the count
//     (the sum) crosses is split into bins of its own until it gives a short list, in which the border is bisected by one
//     wave (a whole workgroup spent 12 us a list on barriers).  Bins hold weights as 64-bit integers, whose sums are the
//     same in any order, in units of 2^-(s + E): s = 50 up to 2^13 classes, one less for each doubling, 43 at 2^20; E the
//     octaves that a bin's weights lie below the first class's.  (Units of the first class's weight alone lose what decides in
//     a tail of a million classes of e^-26 each.)  From bin to bin sums are 64-bit floating point; lists have units of
//     2^-(50 + E), cells 2^-50;
//   the answer: sums of the kept weights by cells (four steps of 64 vectors), made by the pass that fills the last border's
//     list where there is one, the cell in which u falls, then the lane, then the class.
//
// Two looks at a row, for its maximum and its class, take 9.4 us at 256 x 65536 bf16 (temperature 0); those that weigh are bound by
// their 64-bit instructions, some 17 a score at 4.8 cycles a wave each, 12 us a pass there.  A row costs 6 to 7 us of one wave's
// work on the list.  512 x 65536 bf16, rows greedy, uncut, top-k, top-p, min-p and all at once by turns: 78 us; one row of
// 131072, top-k 50: 24 us.
#include "scores.h"
#include <cfloat>
#include <type_traits>

namespace {

constexpr double LOG2E = 1.4426950408889634074;
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

// A value that is the same in all lanes, as a scalar: what comes through LDS or a shuffle is none to the compiler, and every
// loop and test on it would be one per lane.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ float uniform(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }
__device__ __forceinline__ u64 uniform(u64 v) { return (u64)uniform((uint32_t)(v >> 32)) << 32 | uniform((uint32_t)v); }
__device__ __forceinline__ double uniform(double v) { return __longlong_as_double((long long)uniform((u64)__double_as_longlong(v))); }
// lane l's value, l the same in all lanes
__device__ __forceinline__ int lane_at(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ u64 lane_at(u64 v, int l) { return (u64)(uint32_t)lane_at((int)(v >> 32), l) << 32 | (uint32_t)lane_at((int)v, l); }
__device__ __forceinline__ double lane_at(double v, int l) { return __longlong_as_double((long long)lane_at((u64)__double_as_longlong(v), l)); }

// Weights relative to the row's maximum.  With a maximum of +inf its classes weigh 1, all others nothing.
struct Weight {
    double xmax, c; bool inf;
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
#pragma unroll
        for (int h = 0; h < N; h += 4) {           // four chains hide the latency; eight want twice the registers
            double y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = ((double)x[h + e] - xmax) * c;
            exp2_64<4>(y, w + h);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// w <= 1 as an integer in units of 2^-s: the low 52 bits of w + 2^(52 - s).  Lists of at most CAP places and cells of at most 2048
// classes have units of 2^-50: their sums stay below 2^62.
__device__ __forceinline__ u64 fixed(double w, double unit) { return (u64)__double_as_longlong(w + unit) & ((1ull << 52) - 1); }
constexpr int FINE = 50;
constexpr double FINE_UNIT = 4.0, FINE_STEP = 1.0 / (1ull << FINE);
__device__ __forceinline__ u64 fine_units(double w) { return (u64)rint(w * (double)(1ull << FINE)); }       // of any w

// The kept set: x > xt, or x == xt and class <= ti.  Tests that run for every score are written without && and ||, which
// become branches: eight nests of them a vector took four times as long as the comparisons.
struct Cut {
    float xt; int ti;
    __device__ __forceinline__ bool operator()(float x, int j) const { return (x > xt) | ((x == xt) & (j <= ti)); }
};

constexpr int CAP = 512;                           // places of a list: eight a lane of one wave

template <int W, int CELLS> struct Shared {
    // Bins, and copies of them: a lane adds to copy lane % COPIES, which has banks of its own, so few or none of a wave's
    // adds meet, whatever the scores.  More bins, shorter lists (1 x 131072 at top-p 0.9: 1600 places with 128, 390 with 512).
    static constexpr int BINS = W == 1 ? 64 : W >= 8 ? 512 : 128, COPIES = W == 1 ? 1 : W >= 8 ? 16 : 32;
    union {
        u64 bins[BINS][COPIES];
        u64 list[CAP];
    };
    union { double sum[CELLS]; u64 units[CELLS]; int count[CELLS]; } cell;
    alignas(16) double total[BINS];
    double all; int redi; uint32_t red[W];
    int pick; double before; Cut cut;
};

// Largest and smallest finite score, and NaN, of raw vectors: as signed integers whose order is that of the scores (bits
// other than the sign turned over where it is set), two a register with bf16.  A NaN is beyond +inf or -inf.
template <typename T> struct Extremes {
    static constexpr bool B = ET<T>::IS_BF16;
    typedef typename std::conditional<B, short, int>::type I;
    typedef typename std::conditional<B, unsigned short, uint32_t>::type UI;
    typedef I IV __attribute__((ext_vector_type(B ? 2 : 1)));
    typedef UI UV __attribute__((ext_vector_type(B ? 2 : 1)));
    static constexpr I MAG = B ? 0x7FFF : 0x7FFFFFFF, INF = B ? 0x7F80 : 0x7F800000, NEG_INF = (I)(~(UI)INF);
    IV hi, lo; UV fin;                             // fin: from the key behind -inf on, -inf itself being the largest
    __device__ __forceinline__ Extremes() : hi((IV)NEG_INF), lo((IV)INF), fin((UV)(UI)~0u) {}
    __device__ __forceinline__ void add(const i32x4& v) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int word = v[q];
            const IV b = __builtin_bit_cast(IV, word), k = b ^ ((b >> (IV)(I)(sizeof(I) * 8 - 1)) & (IV)MAG);
            hi = __builtin_elementwise_max(hi, k);
            lo = __builtin_elementwise_min(lo, k);
            fin = __builtin_elementwise_min(fin, __builtin_bit_cast(UV, k) + (UV)(UI)~(UI)NEG_INF);
        }
    }
    static __device__ __forceinline__ float score(I k) {
        const I b = k ^ ((k >> (sizeof(I) * 8 - 1)) & MAG);
        return __uint_as_float((uint32_t)(UI)b << (B ? 16 : 0));
    }
    __device__ __forceinline__ void join(float& mine, float& low, bool& nan) const {
#pragma unroll
        for (int e = 0; e < (B ? 2 : 1); ++e) {
            nan |= (hi[e] > INF) | (lo[e] < NEG_INF);
            mine = fmaxf(mine, score(hi[e]));
            const I f = (I)(UI)(fin[e] + (UI)(NEG_INF + 1));
            low = fminf(low, ((f > NEG_INF) & (f < INF)) ? score(f) : INFINITY);
        }
    }
};

// One row as its workgroup of W waves sees it: every wave has a contiguous share of the whole vectors, `steps` of them a
// lane.  Cells in the order of the classes: the row's front end, then the waves' runs of CELL steps, then its back end.
template <typename T, int W> struct Row {
    static constexpr int VEC = ET<T>::VEC, G = W * 64, CELL = 4;
    const T* x;
    RowSpan<T> sp;
    int n, tid, lane, wave, steps, first;          // first: this lane's vector of step 0
    float xe;                                      // of the threads below sp.edge

    __device__ __forceinline__ Row(const T* x_, int n_) : x(x_), sp(x_, n_), n(n_), tid(threadIdx.x), lane(threadIdx.x & 63), wave(uniform((int)threadIdx.x >> 6)) {
        steps = (sp.nvec + G - 1) / G;
        first = wave * steps * 64 + lane;
        xe = tid < sp.edge ? load_score(x, sp.edge_at(tid)) : -INFINITY;
    }
    __device__ __forceinline__ bool valid(int i) const { return i < steps && first + i * 64 < sp.nvec; }
    // Vector i, or the last one of the row in the place of one beyond it (use() takes care of it): a load that is not always
    // made is waited for together with all that follow it.  nvec > 0.
    __device__ __forceinline__ i32x4 load(int i) const { return load_vec(x, sp.vec_at(min(first + i * 64, sp.nvec - 1))); }
    __device__ __forceinline__ i32x4 use(int i, const i32x4& v) const { return wave * steps * 64 + i * 64 + 64 > sp.nvec && !valid(i) ? neg_inf_vec<T>() : v; }
    __device__ __forceinline__ int cls(int i, int e) const { return sp.vec_at(first + i * 64) + e; }
    __device__ __forceinline__ int wave_cells() const { return (steps + CELL - 1) / CELL; }
    __device__ __forceinline__ int cells() const { return W * wave_cells() + 2; }
    __device__ __forceinline__ int cell(int i) const { return 1 + wave * wave_cells() + i / CELL; }
    // the cell of class j; the wave by a product: (v + 0.5) / share is at least 0.5 / 32768 away from a whole number
    __device__ __forceinline__ int cell_of(int j) const {
        const int v = (j - sp.head) / VEC, share = steps * 64;
        if (j < sp.head) return 0;
        if (v >= sp.nvec) return cells() - 1;
        const int w = (int)(((float)v + 0.5f) * __builtin_amdgcn_rcpf((float)share));
        return 1 + w * wave_cells() + (v - w * share) / (64 * CELL);
    }
    __device__ __forceinline__ bool ends_cell(int i) const { return i % CELL == CELL - 1 || i == steps - 1; }
    // f(i, vector i); scores beyond the row are -inf.  U loads are under way at a time, each into registers of its
    // own: moving them along would wait for them.  U = 1 where f itself takes longer than a load.
    template <int U, typename F> __device__ __forceinline__ void each_raw(F f) const {
        if (steps == 0) return;
        i32x4 v[U];
#pragma unroll
        for (int d = 0; d < U; ++d) v[d] = load(d);
#pragma unroll 1
        for (int i = 0; i < steps; i += U) {
#pragma unroll
            for (int d = 0; d < U; ++d) {
                const i32x4 w = use(i + d, v[d]);
                v[d] = load(i + d + U);
                if (i + d < steps) f(i + d, w);
            }
        }
    }
    // f(i, scores of vector i)
    template <int U, typename F> __device__ __forceinline__ void each(F f) const {
        each_raw<U>([&](int i, const i32x4& v) { float s[VEC]; unpack16<T>(v, s); f(i, s); });
    }
    // f(i, scores of vector i) for the steps of cell c, by the wave that has it, until f says stop
    template <typename F> __device__ __forceinline__ void in_cell(int c, F f) const {
        const int wc = wave_cells();
        if (c < 1 || c > W * wc || (c - 1) / wc != wave) return;
        const int i0 = (c - 1) % wc * CELL;
#pragma unroll 1
        for (int i = i0; i < i0 + CELL && i < steps; ++i) {
            float s[VEC];
            unpack16<T>(use(i, load(i)), s);
            if (f(i, s)) return;
        }
    }
};

// Largest v in [lo, hi] with enough(v), which holds at lo.
template <typename F> __device__ __forceinline__ uint32_t last_enough(uint32_t lo, uint32_t hi, F enough) {
#pragma unroll 1
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if (enough(mid)) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// How many of `ties` equal weights `one` the sum needs to get from `over` to target: at least one, at most all.
__device__ __forceinline__ int ties_needed(double over, double one, double target, int ties) {
    if (one == 0 || over + one >= target) return one == 0 ? ties : 1;
    const double m = ceil((target - over) / one);
    return m < (double)ties ? (int)m : ties;
}

// At most CAP places, held by one wave: steps of 64 that hold nothing are skipped.
template <typename T> struct List {
    static constexpr int R = CAP / 64, SHIFT = ET<T>::IS_BF16 ? 16 : 0;    // bits of a key that carry nothing
    const Weight& weight;
    int c, n;                                      // places; classes of the row
    u64 lp[R], lw[R];                              // place (0: none) and weight in units of 2^-(FINE + E)
    int E;
    uint32_t lo, hi, under;                        // smallest and largest key; bit i: weight i is less than min_p
    __device__ __forceinline__ List(const u64* list, int c_, int n_, const Weight& w_, double least, int E_) : weight(w_), c(c_), n(n_), E(E_) {
        const int lane = threadIdx.x & 63;
        float x[R];
        double w[R];
        uint32_t l = 0, h = 0;                     // ~ of the smallest key, the largest
        under = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            lp[i] = lane + 64 * i < c ? list[lane + 64 * i] : 0;
            x[i] = lp[i] ? place_score(lp[i]) : -INFINITY;
            if (lp[i]) { l = max(l, ~key(lp[i])); h = max(h, key(lp[i])); }
        }
        weight.template many<R>(x, w);
#pragma unroll
        for (int i = 0; i < R; ++i) under |= w[i] < least ? 1u << i : 0u;
        if (E) {
#pragma unroll
            for (int i = 0; i < R; ++i) w[i] = ldexp(w[i], E);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) lw[i] = listed(w[i]);
        lo = ~wave_max(l);
        hi = wave_max(h);
    }
    // At least one unit for what weighs anything: u = 0 answers the first kept class, however light it is.
    static __device__ __forceinline__ u64 listed(double w) { const u64 f = fixed(w, FINE_UNIT); return f ? f : w > 0 ? 1 : 0; }
    template <typename P> __device__ __forceinline__ int count(P pred) const {
        int m = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) if (64 * i < c) m += __popcll(__ballot(pred(lp[i])));
        return m;
    }
    template <typename P> __device__ __forceinline__ u64 mass(P pred) const {
        u64 m = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) if (64 * i < c) m += pred(lp[i]) ? lw[i] : 0;
        return wave_sum(m);
    }
    __device__ __forceinline__ u64 all() const { return mass([](u64) { return true; }); }
    static __device__ __forceinline__ uint32_t key(u64 e) { return (uint32_t)(e >> (32 + SHIFT)); }
    // The border among the entries of key v: enough(place) says whether the entries up to a place are.
    template <typename F> __device__ __forceinline__ Cut border_at(uint32_t v, const Cut& was, F enough) const {
        const u64 first = (u64)(ET<T>::IS_BF16 ? v << 16 | ((v & 0x8000u) ? 0u : 0xFFFFu) : v) << 32;
        Cut to = {place_score(first), n};
        if (count([&](u64 e) { return (e ^ first) >> 32 == 0; }) > 1)
            to.ti = (int)~last_enough(~(uint32_t)(n - 1), ~0u, [&](uint32_t mid) { return enough(first | mid); });
        if (to.xt == was.xt) to.ti = min(to.ti, was.ti);
        return to;
    }
    __device__ __forceinline__ Cut cut_count(int k, const Cut& was) const {
        auto enough = [&](u64 from) { return count([&](u64 e) { return e >= from; }) >= k; };
        return border_at(last_enough(lo, hi, [&](uint32_t mid) { return enough((u64)mid << (32 + SHIFT)); }), was, enough);
    }
    // The place at which the mass `need` is reached.  Bisected only until at most 32 entries are left, which are
    // then compared one by one (32 bits of a key to the end: 64 x 400 float32, top-p 0.9: 13.4 us instead of 15.2).  Overwrites list.
    __device__ __forceinline__ Cut cut_mass(u64 need, const Cut& was, u64* list) const {
        const int lane = threadIdx.x & 63;
        uint32_t l = lo, h = hi;
        int left = c, beyond = 0;                  // entries with keys from l on, and beyond h; the mass of the latter
        u64 m_beyond = 0;
#pragma unroll 1
        while (l < h && left - beyond > 32) {
            const uint32_t mid = l + (h - l + 1) / 2;
            u64 m = 0;
            int k = 0;
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (64 * i < c) {
                    const bool in = key(lp[i]) >= mid;
                    m += in ? lw[i] : 0;
                    k += __popcll(__ballot(in));
                }
            m = wave_sum(m);
            if (m >= need) { l = mid; left = k; } else { h = mid - 1; beyond = k; m_beyond = m; }
        }
        if (l == h) return border_at(l, was, [&](u64 from) { return mass([&](u64 e) { return e >= from; }) >= need; });
        int at = 0;
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (64 * i < c) {
                const bool in = lp[i] && key(lp[i]) >= l && key(lp[i]) <= h;
                const u64 b = __ballot(in);
                if (in) { const int to = at + lanes_below(b); list[to] = lp[i]; list[CAP / 2 + to] = lw[i]; }
                at += __popcll(b);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
        const u64 e = lane < at ? list[lane] : 0, f = lane < at ? list[CAP / 2 + lane] : 0;
        u64 front = m_beyond;
#pragma unroll 1
        for (int i = 0; i < at; i += 4) {
#pragma unroll
            for (int d = 0; d < 4; ++d) front += lane_at(e, i + d) > e ? lane_at(f, i + d) : 0;      // lanes from `at` on hold 0
        }
        const u64 hit = __ballot(e && front < need && front + f >= need);
        const u64 last = lane_at(e, hit ? __ffsll(hit) - 1 : 0);
        Cut to = {place_score(last), place_class(last)};
        if (to.xt == was.xt) to.ti = min(to.ti, was.ti);
        return to;
    }
    __device__ __forceinline__ void keep(const Cut& cut) {
        const u64 last = place(score_key(cut.xt), cut.ti);
#pragma unroll
        for (int i = 0; i < R; ++i) if (lp[i] < last) lp[i] = lw[i] = 0;
    }
    __device__ __forceinline__ void drop_under() {
#pragma unroll
        for (int i = 0; i < R; ++i) if (under >> i & 1) lw[i] = 0;
    }
    template <typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int i = 0; i < R; ++i) if (64 * i < c && lw[i]) f(place_class(lp[i]), (lw[i] + ((1ull << E) >> 1)) >> E);       // in cells' units
    }
    // The answer, from entries that are all there is (E = 0): the first class, in the order of the classes, at
    // which the running mass exceeds u times all of it.
    template <typename A> __device__ __forceinline__ void draw(float u, A answer) const {
        const u64 sum = all(), most = (u64)floor((double)u * (double)sum);             // a running mass > most
        // lower classes are larger ~class: the largest one down from which more than `most` has gathered
        const uint32_t who = last_enough(~(uint32_t)(n - 1), ~0u, [&](uint32_t mid) { return mass([&](u64 e) { return (uint32_t)e >= mid; }) > most; });
        float x = -INFINITY;
#pragma unroll
        for (int i = 0; i < R; ++i) if (64 * i < c && lw[i] && (uint32_t)lp[i] == who) x = place_score(lp[i]);
        if (x > -INFINITY) answer((int)~who, weight(x), (double)sum * FINE_STEP);
    }
};

// A list of at most 64 places, one a lane, compared with each other one by one.
template <typename T, typename A> __device__ __forceinline__ void draw_short(const u64* list, int c, int k, float p, double least, float u, const Weight& weight, A answer) {
    const int lane = threadIdx.x & 63;
    const u64 e = lane < c ? list[lane] : 0;
    const double w = lane < c ? weight(place_score(e)) : 0.0;
    u64 f = List<T>::listed(w);
    if (k < c || p < 1.f) {
        u64 above = 0;                             // mass and number of the entries in front of this one
        int rank = 0;
#pragma unroll 1
        for (int i = 0; i < c; i += 4) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {          // lanes from c on hold 0
                const bool front = lane_at(e, i + d) > e;
                above += front ? lane_at(f, i + d) : 0;
                rank += front;
            }
        }
        if (rank >= k) f = 0;
        if (p < 1.f && above >= (u64)ceil((double)p * (double)wave_sum(f))) f = 0;
    }
    if (w < least) f = 0;
    const u64 sum = wave_sum(f), most = (u64)floor((double)u * (double)sum);
    u64 before = 0;                                // mass of the kept entries of lower classes
#pragma unroll 1
    for (int i = 0; i < c; i += 4) {
#pragma unroll
        for (int d = 0; d < 4; ++d) before += (uint32_t)lane_at(e, i + d) > (uint32_t)e ? lane_at(f, i + d) : 0;
    }
    if (before <= most && most < before + f) answer(place_class(e), w, (double)sum * FINE_STEP);
}

template <typename T, int W, int CELLS>
__global__ __launch_bounds__(W * 64, 4) void sample_kernel(SampleArgs a) {
    typedef Row<T, W> R;
    typedef Shared<W, CELLS> S;
    constexpr int VEC = R::VEC, G = R::G, BINS = S::BINS;
    __shared__ S sh;
    const size_t r = blockIdx.x;
    const R row((const T*)((const char*)a.x + r * a.stride * ET<T>::ES), a.n);
    const int tid = row.tid, lane = row.lane, wave = row.wave, n = a.n;
    const float u = a.u[r], t = a.tp ? a.tp[r] : a.t, p = a.pp ? a.pp[r] : a.p, q = a.qp ? a.qp[r] : a.q;
    int k = a.kp ? a.kp[r] : a.k;
    auto fixed_answer = [&](int label, float lp) { a.labels[r] = label; a.logp[r] = lp; };                 // by one thread
    auto answer = [&](int label, double w, double all) { fixed_answer(label, (float)ln_64(w / all)); };

    auto block_max = [&](uint32_t v) {
        v = wave_max(v);
        if constexpr (W == 1) return v;
        __syncthreads();
        if (lane == 0) sh.red[wave] = v;
        __syncthreads();
        return wave_max(lane < W ? sh.red[lane] : 0u);
    };
    // the row's maximum, its smallest finite score, and whether a NaN is there
    float mine = row.xe, low = row.xe > -INFINITY ? row.xe : INFINITY;
    bool nan = row.xe != row.xe;
    {
        Extremes<T> x;
        row.template each_raw<4>([&](int i, const i32x4& v) { x.add(v); });
        if (row.steps) x.join(mine, low, nan);
    }
    const uint32_t top = block_max(nan ? KEY_NAN : score_key(mine));
    if (top == KEY_NAN || !(t >= 0.f) || !(t < INFINITY) || k < 0 || !(p > 0.f) || !(p <= 1.f) || !(q >= 0.f) || !(q <= 1.f) || !(u >= 0.f) || !(u < 1.f)) {
        if (tid == 0) fixed_answer(-1, NAN);
        return;
    }
    if (top == KEY_NEG_INF) { if (tid == 0) fixed_answer(-1, -INFINITY); return; }
    const float xmax = key_score(top);
    const Weight weight = {(double)xmax, t > 0.f ? LOG2E / (double)t : 0.0, xmax == INFINITY};
    // Bins have units of 2^-(s + E), E the octaves that all weights of a bin lie below the first one: n of at most 2^s are at most 2^63.
    const double bin_unit = (double)(1ull << (52 - min(50, 31 + __clz(n - 1))));
    if (t == 0.f || k == 1) {
        int at = n;
        row.template each<4>([&](int i, const float* s) {
#pragma unroll
            for (int e = VEC - 1; e >= 0; --e) if (s[e] == xmax) at = min(at, row.cls(i, e));
        });
        if (tid < row.sp.edge && row.xe == xmax) at = min(at, row.sp.edge_at(tid));
        at = (int)~block_max(~(uint32_t)at);
        if (tid == 0) fixed_answer(at, 0.f);
        return;
    }
    if (k == 0 || k > n) k = n;

    // min_p: a weight is only computed where a 32-bit estimate of the border, with room, says that it may pass
    const double least = q > 0.f ? (double)q : 0.0;
    const float xq = q > 0.f && !weight.inf ? (float)((double)xmax + (double)(__builtin_amdgcn_logf(q) - 1e-3f) / weight.c) : -INFINITY;
    const float xlow = xq - fabsf(xq) * 1e-6f;

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
            for (int e = 0; e < VEC; ++e) x[e] = ((s[e] == cut.xt) & (row.cls(i, e) > cut.ti)) ? -INFINITY : x[e];
        }
        return true;
    };
    // counts by cells of the scores that pass, as prefix sums: cell.count[c] = how many lie in front of cell c.  Returns all.
    auto count_cells = [&](auto pred) {
        __syncthreads();
        const int cells = row.cells();
        int m = 0;
        row.template each<2>([&](int i, const float* s) {
            const bool ok = row.valid(i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) m += __popcll(__ballot(ok & pred(s[e], row.cls(i, e))));
            if (row.ends_cell(i)) { if (lane == 0) sh.cell.count[row.cell(i)] = m; m = 0; }
        });
        if (wave == 0) {
            const u64 b = __ballot(tid < row.sp.edge && pred(row.xe, row.sp.edge_at(tid))), front = (1ull << row.sp.head) - 1;
            if (lane == 0) { sh.cell.count[0] = __popcll(b & front); sh.cell.count[cells - 1] = __popcll(b & ~front); }
        }
        __syncthreads();
        if (wave == 0) {
            int run = 0;
#pragma unroll 1
        for (int c = 0; c < cells; c += 64) {
                const int m = c + lane < cells ? sh.cell.count[c + lane] : 0;
                const int s = wave_scan(m);
                if (c + lane < cells) sh.cell.count[c + lane] = run + s - m;
                run += lane_at(s, 63);
            }
            if (lane == 0) sh.pick = run;
        }
        __syncthreads();
        return uniform(sh.pick);
    };
    // The kept scores in [xa, xb], xa > -inf, as places in the list (in no particular order: everything that is made of it is
    // a set, or a sum of integers).  Returns how many there are; more than CAP are not all in it.  Few scores pass, so what
    // counts is the test, two instructions a score, and that a lane with a hit handles it alone.  With sum, the weights of the
    // scores beyond xb that min_p leaves are added up by cells, in integer units.
    auto collect = [&](float xa, const float xb, bool sum) {
        __syncthreads();
        if (tid == 0) sh.pick = 0;
        __syncthreads();
        xa = fmaxf(xa, cut.xt);
        if (xa > xb) return 0;
        auto append = [&](float x, int j) {
            if (cut.ti < n && x == cut.xt && j > cut.ti) return;
            const int at = atomicAdd(&sh.pick, 1);
            if (at < CAP) sh.list[at] = place(score_key(x), j);
        };
        double cell_sum = 0;
        row.template each<2>([&](int i, const float* s) {
            u64 some = 0;
#pragma unroll
            for (int e = 0; e < VEC; ++e) some |= __ballot(__builtin_amdgcn_fmed3f(s[e], xa, xb) == s[e]);
            if (some) {
                uint32_t in = 0;
#pragma unroll
                for (int e = 0; e < VEC; ++e) in |= __builtin_amdgcn_fmed3f(s[e], xa, xb) == s[e] ? 1u << e : 0u;
                while (in) {
                    const int e = __ffs(in) - 1;
                    in &= in - 1;
                    float x = s[0];
#pragma unroll
                    for (int o = 1; o < VEC; ++o) x = e == o ? s[o] : x;
                    append(x, row.cls(i, e));
                }
            }
            if (sum) {
                float x[VEC];
                bool any = false;
#pragma unroll
                for (int e = 0; e < VEC; ++e) { const bool k = (s[e] > xb) & (s[e] >= xlow); x[e] = k ? s[e] : -INFINITY; any |= k; }
                if (__ballot(any)) {
                    double w[VEC];
                    weight.template many<VEC>(x, w);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) cell_sum += w[e] >= least ? w[e] : 0.0;
                }
                if (row.ends_cell(i)) {
                    cell_sum = wave_sum(cell_sum);
                    if (lane == 0) sh.cell.units[row.cell(i)] = fine_units(cell_sum);
                    cell_sum = 0;
                }
            }
        });
        if (tid < row.sp.edge && row.xe >= xa && row.xe <= xb) append(row.xe, row.sp.edge_at(tid));
        __syncthreads();
        const int c = uniform(sh.pick);
        __syncthreads();
        return c;
    };
    // The class of the m-th one, by class, of the scores equal to x.
    auto nth = [&](float x, int m) {
        auto is = [&](float s, int) { return s == x; };
        count_cells(is);
        if (wave == 0) {                           // the last cell with fewer than m in front of it
            int c = 0;
#pragma unroll 1
            for (int b = 0; b < row.cells(); b += 64) {
                const bool in = b + lane < row.cells() && sh.cell.count[b + lane] < m;
                c += __popcll(__ballot(in));
            }
            if (lane == 0) sh.pick = c - 1;
        }
        __syncthreads();
        const int c = uniform(sh.pick), cells = row.cells();
        int left = m - uniform(sh.cell.count[c]);           // the left-th one of that cell
        row.in_cell(c, [&](int i, const float* s) {
            int own = 0;
            const bool ok = row.valid(i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) own += ok && s[e] == x ? 1 : 0;
            const int s0 = wave_scan(own), here = lane_at(s0, 63);
            if (here < left) { left -= here; return false; }
            if (s0 - own < left && left <= s0) {
                int rank = s0 - own;
#pragma unroll
                for (int e = 0; e < VEC; ++e) if (s[e] == x && ++rank == left) sh.redi = row.cls(i, e);
            }
            return true;
        });
        if (wave == 0 && (c == 0 || c == cells - 1)) {
            const u64 b = __ballot(tid < row.sp.edge && row.xe == x), front = (1ull << row.sp.head) - 1, here = c == 0 ? b & front : b & ~front;
            if ((here >> lane & 1) && lanes_below(here) == left - 1) sh.redi = row.sp.edge_at(tid);
        }
        __syncthreads();
        const int j = uniform(sh.redi);
        __syncthreads();
        return j;
    };
    // A key that k of the threads' maxima reach, to 16 bits (bisected by one wave).
    auto bound = [&] {
        uint32_t* maxima = (uint32_t*)sh.bins;
        maxima[tid] = score_key(mine) >> 16;
        __syncthreads();
        if (wave == 0) {
            uint32_t m[W];
#pragma unroll
            for (int w = 0; w < W; ++w) m[w] = maxima[w * 64 + lane];
            const uint32_t v = last_enough(0, top >> 16, [&](uint32_t mid) {
                int s = 0;
#pragma unroll
                for (int w = 0; w < W; ++w) s += __popcll(__ballot(m[w] >= mid));
                return s >= k;
            });
            if (lane == 0) sh.pick = (int)(v << 16);
        }
        __syncthreads();
        return uniform((uint32_t)sh.pick);
    };

    // ---- borders ----------------------------------------------------------------------------------------------------
    // The kept scores with keys in [klo, khi] by bins, and what each weighs (mass) or counts: bins of the distance to the first
    // score, or (shift >= 0) of the keys down from khi.
    uint32_t klo = 0, khi = top;
    float scale = 0;
    int per_octave = 31;                           // 2^per_octave bins of the distance lie within an octave of the weight, or more
    int octaves = 0;                               // that the weights from khi down lie below the first one
    auto upper_score = [](uint32_t k) { return key_score(k == 0x7FFFFFFFu ? k - 1 : k); };  // no score has the key of -0, and as a number it is 0
    auto fill_bins = [&](bool mass, int shift) {
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < S::COPIES * BINS; i += G) (&sh.bins[0][0])[i] = 0;
        __syncthreads();
        const float xlo = klo ? key_score(klo) : -INFINITY, xhi = upper_score(khi);
        // a count is a sum of weights of 1 in units of 1
        const int eb = mass && shift < 0 ? per_octave : 31, unit0 = __double2hiint(mass ? bin_unit : 4503599627370496.0) - (octaves << 20);
        auto unit = [&](int b) { return __hiloint2double(__mul24(b >> eb, -(1 << 20)) + unit0, 0); };       // 2^-(b >> eb)
        auto drop = [&](float x, double w) {
            if (x > xhi) return;
            const int b = shift < 0 ? (int)fminf((xmax - x) * scale, (float)(BINS - 1)) : (int)((khi - score_key(x)) >> shift);
            atomicAdd(&sh.bins[b][lane & (S::COPIES - 1)], fixed(w, unit(b)));
        };
        row.template each<1>([&](int i, const float* s) {
            float x[VEC];
            if (!only_kept(i, s, x, xlo)) return;
            double w[VEC];
            if (mass) weight.template many<VEC>(x, w);
            else {
                const double one = row.valid(i) ? 1.0 : 0.0;
#pragma unroll
                for (int e = 0; e < VEC; ++e) w[e] = one;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) if (s[e] >= xlo) drop(s[e], w[e]);
        });
        if (tid < row.sp.edge && row.xe >= xlo && cut(row.xe, row.sp.edge_at(tid))) drop(row.xe, mass ? weight(row.xe) : 1.0);
        __syncthreads();
#pragma unroll 1
        for (int b = tid; b < BINS; b += G) {
            u64 s = 0;
#pragma unroll 8
            for (int i = 0; i < S::COPIES; ++i) s += sh.bins[b][(i + tid) & (S::COPIES - 1)];
            sh.total[b] = (double)s * (unit(b) * 2.2204460492503131e-16);           // 2^-52
        }
        __syncthreads();
    };
    // Sum of the bins; the first bin at which the running sum, from `above` on, reaches target, or the last one that holds anything
    // if rounding leaves none (every wave, BINS / 64 bins a lane, the same sums in the same order).
    constexpr int BL = BINS / 64;
    auto bin_sum = [&]() {
        double s = 0;
#pragma unroll
        for (int i = 0; i < BL; ++i) s += sh.total[BL * lane + i];
        return wave_sum(s);
    };
    auto bin_reach = [&](double target, double& above) {
        double own = 0;
#pragma unroll
        for (int i = 0; i < BL; ++i) own += sh.total[BL * lane + i];
        const double s = wave_scan(own);
        const u64 some = __ballot(own > 0), hit = __ballot(own > 0 && above + s >= target);
        const int l = hit ? __ffsll(hit) - 1 : some ? 63 - __clzll(some) : 0;
        double run = above + lane_at(s - own, l);
        int b = BL * l;
#pragma unroll 1
        for (int i = 0; i < BL; ++i) {
            const double v = uniform(sh.total[BL * l + i]);
            if (v > 0) { b = BL * l + i; above = run; if (run + v >= target) break; }
            run += v;
        }
        return b;
    };
    // the last key up to top with holds(score), which holds for -inf and below: 64 keys tried at a time
    auto last_key = [&](auto holds) {
        uint32_t lo = KEY_NEG_INF, hi = top;
#pragma unroll 1
        while (lo < hi) {
            const uint32_t step = (hi - lo) / 64 + 1, key = lo + lane * step;
            const int m = __popcll(__ballot((lane == 0) | ((key > lo) & (key <= hi) & holds(key_score(min(max(key, lo), hi))))));
            const uint32_t from = lo + (m - 1) * step;
            hi = min(hi, from + (step - 1));
            lo = from;
        }
        return lo;
    };

    // Pass 0: rows that fit in a list, and top_k of which the threads' maxima give one; the list is all there is.
    // Pass 1: the border of top_k, pass 2: the border of top_p.  Bins; then the bin that the border is in, split by keys until
    // it holds a list or one key.  The last of the two also adds up what is kept for certain.  One loop, so that there is one
    // copy of everything (written out for each use the code was 87 KB, more than the instruction cache holds).
    bool summed = false;                           // the cells hold what is kept, in integer units
#pragma unroll 1
    for (int pass = 0; pass < (W == 1 ? 1 : 3); ++pass) {
        const bool mass = pass == 2, sum = (mass || (pass == 1 && !(p < 1.f))) && u > 0.f;       // at u = 0 less than a unit counts
        double above = 0, target = (double)k;
        int shift = -1, c;
        if (pass == 0) {
            klo = KEY_NEG_INF + 1;                 // -inf weighs nothing: never in the list
            if (W > 1 && n > CAP) {
                if (k > G / 2) continue;
                klo = bound();
                if (klo <= KEY_NEG_INF) continue;
            }
            khi = top;
        } else {
            if (mass ? !(p < 1.f) : k == n) continue;
            klo = 0; khi = top; octaves = 0;
            // BINS over 32 octaves of the weight, or finer where the row is narrower
            const float smallest = key_score(~block_max(~score_key(low)));
            scale = (float)fmin(BINS / 32 * weight.c, 1e30);
            if ((xmax - smallest) * scale < (float)(BINS - 1) && xmax > smallest) scale = (float)(BINS - 1) / (xmax - smallest);
            const float bins = (float)((double)scale / weight.c);
            per_octave = weight.inf || !(bins < 1e9f) ? 31 : bins > 1.001f ? ilogbf(0.999f * bins) + 1 : 0;
        }
#pragma unroll 1
        for (;;) {
            if (pass) {
                fill_bins(mass, shift);
                if (mass && shift < 0) target = (double)p * bin_sum();
                const int b = bin_reach(target, above);
                if (mass && shift < 0) octaves = min(50, b >> per_octave);
                if (shift < 0) {                   // from the first key that is not beyond the bin to the last that has reached it
                    khi = last_key([&](float x) { return !((xmax - x) * scale < (float)b); });
                    klo = b == BINS - 1 ? KEY_NEG_INF + 1 : max(KEY_NEG_INF, last_key([&](float x) { return !((xmax - x) * scale < (float)(b + 1)); })) + 1;
                } else {
                    khi -= (uint32_t)b << shift;
                    klo = khi - min(khi - klo, (1u << shift) - 1);
                }
            }
            c = collect(key_score(klo), upper_score(khi), sum);
            if (!pass || c <= CAP || klo >= khi) break;
            shift = 0;                             // every round leaves 2 / BINS of the keys
            while ((khi - klo) >> shift >= (uint32_t)BINS) ++shift;
        }
        if (pass == 0 && c > CAP) continue;
        if (pass == 1 && target > above + (double)c) continue;                     // top_k reaches into scores of -inf: all others are kept
        if (c <= CAP) {
            if (wave == 0) {
                if (!pass && c <= 64) { draw_short<T>(sh.list, c, k, p, least, u, weight, answer); return; }
                List<T> list(sh.list, c, n, weight, least, octaves);
                if (pass ? !mass : k < c) { cut = list.cut_count((int)(target - above), cut); list.keep(cut); }
                if (pass ? mass : p < 1.f) {
                    // what the bins' rounding says more than the list holds is all of it
                    const u64 all = list.all();
                    const double need = pass ? ldexp(target - above, FINE + list.E) : (double)p * (double)all;
                    cut = list.cut_mass(need < (double)all ? max((u64)1, (u64)ceil(need)) : all, cut, sh.list);
                    list.keep(cut);
                }
                list.drop_under();
                if (!pass) { list.draw(u, answer); return; }
                if (sum) list.each([&](int j, u64 w) { const int at = row.cell_of(j); if (at > 0 && at < row.cells() - 1) atomicAdd(&sh.cell.units[at], w); });
                if (lane == 0) sh.cut = cut;
            }
            if (!pass) return;
            __syncthreads();
            cut = {uniform(sh.cut.xt), uniform(sh.cut.ti)};
            summed = sum;
        } else {                                   // c equal scores
            const float x = key_score(khi);
            const int need = mass ? ties_needed(above, weight(x), target, c) : (int)(target - above);
            if (x > -INFINITY) cut = {x, need < c ? nth(x, need) : x == cut.xt ? cut.ti : n};           // -inf weighs nothing: no cut
        }
    }
    if constexpr (W == 1) return;                  // one wave: rows that fit in a list
    // ---- the answer -------------------------------------------------------------------------------------------------
    auto share = [&](float x, int j) {             // the weight of a class that is kept, else 0
        double w = 0;
        if ((x >= xlow) & cut(x, j)) { w = weight(x); if (w < least) w = 0; }
        return w;
    };
    // weights of a vector's kept scores; false: there are none in the wave
    auto shares = [&](int i, const float* s, double* w) {
        float x[VEC];
        if (!only_kept(i, s, x, xlow)) return false;
        weight.template many<VEC>(x, w);
        if (least > 0) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) w[e] = w[e] >= least ? w[e] : 0.0;
        }
        return true;
    };
    __syncthreads();
    auto set_cell = [&](int c, double s) { if (summed) sh.cell.units[c] = fine_units(s); else sh.cell.sum[c] = s; };
    auto cell_at = [&](int c) { return summed ? (double)sh.cell.units[c] * FINE_STEP : sh.cell.sum[c]; };
    double cell_sum = 0;
    if (!summed) row.template each<1>([&](int i, const float* s) {
        double w[VEC];
        if (shares(i, s, w)) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) cell_sum += w[e];
        }
        if (row.ends_cell(i)) {
            cell_sum = wave_sum(cell_sum);
            if (lane == 0) sh.cell.sum[row.cell(i)] = cell_sum;
            cell_sum = 0;
        }
    });
    const int cells = row.cells();
    if (wave == 0) {
        const double w = tid < row.sp.edge ? share(row.xe, row.sp.edge_at(tid)) : 0.0;
        const double f = wave_sum(tid < row.sp.head ? w : 0.0), b = wave_sum(tid < row.sp.head ? 0.0 : w);
        if (lane == 0) { set_cell(0, f); set_cell(cells - 1, b); }
    }
    __syncthreads();
    double all = 0;
    if (wave == 0) {
#pragma unroll 1
        for (int c = 0; c < cells; c += 64) all += wave_sum(c + lane < cells ? cell_at(c + lane) : 0.0);
        const double target = (double)u * all;
        // the first cell whose running sum exceeds the target, or the last one that holds anything
        double run = 0, found_before = 0;
        int found = -1, last = 0; double last_before = 0;
#pragma unroll 1
        for (int c = 0; c < cells; c += 64) {
            const double m = c + lane < cells ? cell_at(c + lane) : 0.0;
            const double s = wave_scan(m);
            const u64 hit = __ballot(m > 0 && run + s > target), some = __ballot(m > 0);
            if (some) { const int l = 63 - __clzll(some); last = c + l; last_before = run + lane_at(s - m, l); }
            if (hit) { const int l = __ffsll(hit) - 1; found = c + l; found_before = run + lane_at(s - m, l); break; }
            run += lane_at(s, 63);
        }
        if (lane == 0) { sh.pick = found >= 0 ? found : last; sh.before = found >= 0 ? found_before : last_before; sh.all = all; }
    }
    __syncthreads();
    const int at = uniform(sh.pick);
    const double before = uniform(sh.before);
    all = uniform(sh.all);
    const double target = (double)u * all;
    // the class within the cell: the lane in which the running sum exceeds the target, then its element; the last one that
    // weighs anything if rounding leaves none
    double run = before;
    int last = -1; double last_w = 0;
    row.in_cell(at, [&](int i, const float* s) {
        double w[VEC];
        if (!shares(i, s, w)) return false;
        double own = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) own += w[e];
        const double p = wave_scan(own);
        const u64 hit = __ballot(own > 0 && run + p > target);
        double front = run + (p - own);
        int mine = -1, lastc = -1; double mw = 0, lastw = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            front += w[e];
            if (w[e] > 0) {
                lastc = row.cls(i, e); lastw = w[e];
                if (mine < 0 && front > target) { mine = lastc; mw = lastw; }
            }
        }
        if (mine < 0) { mine = lastc; mw = lastw; }
        if (hit) {
            if (lane == __ffsll(hit) - 1) answer(mine, mw, all);
            last = -1;
            return true;
        }
        const u64 some = __ballot(own > 0);
        if (some) { const int l = 63 - __clzll(some); last = lane_at(lastc, l); last_w = lane_at(lastw, l); }
        run += lane_at(p, 63);
        return false;
    });
    if (lane == 0 && last >= 0) answer(last, last_w, all);
    if (wave == 0 && (at == 0 || at == cells - 1)) {
        const bool here = tid < row.sp.edge && (tid < row.sp.head) == (at == 0);
        const int j = here ? row.sp.edge_at(tid) : 0;
        const double w = here ? share(row.xe, j) : 0.0;
        const double p = wave_scan(w);
        const u64 hit = __ballot(w > 0 && before + p > target), some = __ballot(w > 0);
        if (lane == (hit ? __ffsll(hit) - 1 : 63 - __clzll(some))) answer(j, w, all);
    }
}

template <typename T> void launch(const SampleArgs& a, int rows, hipStream_t s) {
    constexpr int VEC = ET<T>::VEC;
    const int nv = a.n / VEC;
    // Waves a row: few rows have the chip to themselves, many share it.  Top-p 0.9, us with 4 / 8 / 16 waves: 64 x 4000 float32
    // 21.4 / 18.0 / 19.4, 1024 x 4000 32.1 / 43.8 / 73.2, 4096 x 8000 150 / 207 / 338; with 8 / 16: 200 x 40961 49.9 / 45.9,
    // 512 x 65536 bf16 110 / 128, 4096 x 65536 689 / 944.
    if (a.n <= CAP) sample_kernel<T, 1, 2 + (CAP / VEC / 64 + 3) / 4><<<rows, 64, 0, s>>>(a);
    else if (nv <= 512 || (nv <= 2048 && rows > 256)) sample_kernel<T, 4, 10><<<rows, 256, 0, s>>>(a);
    else if (nv <= 2048 || rows > 256) sample_kernel<T, 8, (1 << 20) / VEC / 256 + 10><<<rows, 512, 0, s>>>(a);
    else sample_kernel<T, 16, (1 << 20) / VEC / 256 + 18><<<rows, 1024, 0, s>>>(a);
}

}  // namespace

extern "C" int stgcn_sample_labels(int dtype, const void* logits, size_t row_stride, const float* u, const float* temperatures, float temperature,
                                   const int* top_ks, int top_k, const float* top_ps, float top_p, const float* min_ps, float min_p,
                                   int64_t* labels, float* logp, int rows, int ncls, void* stream) {
    if (!logits || !u || !labels || !logp || rows < 1 || rows >= (1 << 24) || ncls < 1 || ncls > (1 << 20) || row_stride < (size_t)ncls) return STGCN_ERR_ARG;
    SampleArgs a = {logits, row_stride, u, temperatures, top_ks, top_ps, min_ps, temperature, top_k, top_p, min_p, (long long*)labels, logp, ncls};
    if (dtype == STGCN_BF16) launch<bf16>(a, rows, (hipStream_t)stream);
    else if (dtype == STGCN_F32) launch<float>(a, rows, (hipStream_t)stream);
    else return STGCN_ERR_ARG;
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}
