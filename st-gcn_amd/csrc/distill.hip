// Distillation from a teacher's top logits: loss and gradient over rows of class scores.
//
// One row: student scores x[0..n), the teacher's listed classes i_1..i_K with scores t_k (i_k < 0: absent), rho = log of
// the teacher's unlisted mass at temperature T (absent: -inf).  With z = x / T
//   A = log(sum_k e^{t_k/T} + e^rho),  p_k = e^{t_k/T - A},  p_r = e^{rho - A}
//   S_l, S_r = sum of e^z over the listed classes and over the others,  S = S_l + S_r
//   KL = sum_k p_k (log p_k - z_{i_k} + log S) + p_r (log p_r - log S_r + log S)
//   loss = (1 - w) T^2 KL + w (log sum_j e^{x_j} - x_y)
//   d loss / d x_j = (1 - w) T e^{z_j} (1/S - [j not listed] p_r/S_r) - (1 - w) T sum_{k: i_k = j} p_k
//                    + w (e^{x_j} / sum e^x - [j = y])
// S_r is summed without the listed classes (a bit map of the row in LDS) instead of as S - S_l: a teacher whose list
// carries nearly all of the mass would leave nothing of the difference but rounding.  It stays relative to its own largest
// score m, as do the gradients of its classes: with M the row's largest score and a = e^{(m - M)/T}, the gradient of a class
// that is not listed is (1 - w) T e^{(x - m)/T} (a/S' - p_r/S_r'), S' relative to M, S_r' to m.  Relative to M, e^z of all of
// them is 0 in 32 bits from a gap of 87 T on, and p_r with it.
//
// Bound by memory where rows are wide: loss and gradient in one pass with the row in registers move what a copy moves, at a
// copy's rate (8192 x 65536 bf16, 405 us, 5.3 TB/s).  Narrow rows are bound by what a row costs whatever its width, so four
// share a wave (16384 x 400 float32: 20 us, of 6 to 10 for the bytes).
#include "scores.h"
#include "listed_map.h"

namespace {

constexpr int MAX_K = 256;
constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.6931471805599453094;

// What a row's forward leaves for its gradient: the largest score xl of the row, which listed classes are relative to, the
// largest xr of those that are not listed, which these are relative to, and the factors g of e^{./T} and h of e^. on either
// side.  xl is NaN for a row whose gradient is zero whatever it holds.
struct RowStats { float xl, xr, gl, gr, hl, hr; };

struct DistillArgs {
    const void* x; size_t stride;
    const float* val; const long long* idx; const float* rest; const long long* labels;
    double* loss_rows; float* loss; RowStats* stats; float* probs;
    void* dx; float scale;                     // of the gradient, where it is written
    int rows, n, k;
    float c, c1, fp, w1;                       // log2(e) / T, log2(e), (1 - w) T, w
    double T, invT, w;
};

// Waves that work on one row: W of them, and for W = 1 several rows share a workgroup and no barrier is needed.
template <int W> __device__ __forceinline__ void group_sync() {
    if constexpr (W == 1) { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier(); }
    else __syncthreads();
}

// ---- the teacher's side of a row, the work of one group of L lanes (scores.h) ---------------------------------------------------------------------
// Entries in LDS: class (-1: none, or a class that an earlier entry has), the student's score there, and the share p (with
// duplicates their sum; before it is normalised, e^{t/T - max}).  Next to them what the others need: none of it waits for
// the student's maximum or sums.
template <int K> struct Listed {                // K: entries at most
    int cls[K]; float x[K]; double p[K];
    double own, cross, pr;                     // sum of p log p (p_r among them), sum of p (z - the largest listed z), p_r
    double sl, sl1; float xmax;                // sums of 2^{(x - xmax) c} over the listed classes, xmax their maximum
    int flags;                                 // 1: there is a teacher, 2: an entry or the label is out of range
    unsigned char later[K];
};
__device__ __forceinline__ void wave_sync() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier(); }

// The entries as they come from the teacher: read ahead of the row, whose loads then need not be waited for (they return in
// order), and always, the last entry in the place of one beyond it.
template <int L, int K> struct Entries {
    long long i[K / L]; float t[K / L];
    __device__ __forceinline__ void load(const DistillArgs& a, size_t r, int lane) {
#pragma unroll
        for (int c = 0; c < K / L; ++c) {
            const size_t at = r * a.k + min(lane + c * L, a.k - 1);
            i[c] = a.idx[at];
            t[c] = a.val[at];
        }
    }
};

// Classes and student scores of the entries.
template <typename T, int L, int K> __device__ __forceinline__ void listed_load(const DistillArgs& a, const Entries<L, K>& from, const T* x, int lane, Listed<K>& l) {
    bool bad = false, has = false;
    float s[K / L];
#pragma unroll
    for (int c = 0; c < K / L; ++c) s[c] = load_score(x, (size_t)(from.i[c] >= 0 && from.i[c] < a.n ? from.i[c] : 0));
#pragma unroll
    for (int c = 0; c < K / L; ++c) {
        const int e = lane + c * L;
        if (e < a.k) {
            const long long i = from.i[c];
            const float t = from.t[c];
            const bool in = i >= 0 && i < a.n;
            l.cls[e] = in ? (int)i : -1;
            l.x[e] = in ? s[c] : -INFINITY;
            bad |= i >= a.n || (in && !(t < INFINITY));
            const float u = in && t < INFINITY ? t : -INFINITY;
            l.p[e] = (double)u;
            has |= u > -INFINITY;
        }
    }
    const int flags = (group_any<L>(has) && a.w < 1.0 ? 1 : 0) | (group_any<L>(bad) ? 2 : 0);
    if (lane == 0) l.flags = flags;
    wave_sync();
}

// Shares and sums.  `rho` is only looked at where there is an entry.
template <bool TWO, int L, int K> __device__ __forceinline__ void listed_sums(const DistillArgs& a, int lane, float rho32, Listed<K>& l) {
    float tmax = -INFINITY, xmax = -INFINITY;
    for (int e = lane; e < a.k; e += L) { tmax = fmaxf(tmax, (float)l.p[e]); xmax = fmaxf(xmax, l.x[e]); }
    tmax = group_max<L>(tmax); xmax = group_max<L>(xmax);
    int flags = l.flags;
    const bool any = flags & 1;
    if (any && !(rho32 < INFINITY)) flags |= 2;
    // Relative to the larger of t_max / T and rho; the scores' differences are taken before they are divided (a product less its
    // own rounded value is no zero when it becomes one fused operation, and next to T = 1e-16 more than the whole).
    const double invT = a.invT, rho = (double)rho32, over = rho - (double)tmax * invT;
    const bool by_rho = over > 0;
    const double ref = by_rho ? 0.0 : (double)tmax, z0 = by_rho ? -rho : 0.0, zr = by_rho ? 0.0 : over;
    double s = 0, sz = 0, sx = 0;
    float sl = 0.f, sl1 = 0.f;
    for (int e = lane; e < a.k; e += L) {
        const double t = l.p[e];
        const float x = l.x[e];
        double p = 0;
        if (any && t > -INFINITY) {
            const double z = (t - ref) * invT + z0;
            p = exp2_64(z * LOG2E);
            s += p; sz += p * z;
            if (p > 0) sx += p * ((double)x - (xmax > -INFINITY ? (double)xmax : 0.0));
        }
        l.p[e] = p;
        if (l.cls[e] >= 0 && (xmax > -INFINITY || x != x)) {           // a NaN is no maximum, and makes the sums NaN
            sl += exp2_32((x - xmax) * a.c);
            if constexpr (TWO) sl1 += exp2_32((x - xmax) * a.c1);
        }
    }
    s = group_sum<L>(s); sz = group_sum<L>(sz); sx = group_sum<L>(sx);
    const double er = any ? exp2_64(zr * LOG2E) : 0.0;
    s += er;
    const double inv = any ? 1.0 / s : 0.0, ls = any ? ln_64(s) : 0.0;
    for (int e = lane; e < a.k; e += L) l.p[e] *= inv;
    const double pr = er * inv, sl64 = group_sum<L>((double)sl), sl164 = TWO ? group_sum<L>((double)sl1) : 0.0;
    if (lane == 0) {
        l.own = (sz + (er > 0 ? er * zr : 0.0)) * inv - ls;         // sum of p log p = sum of p (z - ln s), all p being 1
        l.cross = sx * inv * (double)a.c * LN2;
        l.pr = pr; l.sl = sl64; l.sl1 = sl164; l.xmax = xmax; l.flags = flags;
    }
    wave_sync();
}

// Entries of one class: the first keeps the sum of their p, the others leave the list; sums are made anew.  Rare.
template <bool TWO, int L, int K> __device__ __forceinline__ void listed_merge(const DistillArgs& a, int lane, Listed<K>& l) {
    for (int e = lane; e < a.k; e += L) {
        bool later = false;
        for (int o = 0; o < e; ++o) later |= l.cls[o] == l.cls[e];
        l.later[e] = later;
    }
    wave_sync();
    float sl = 0.f, sl1 = 0.f;
    for (int e = lane; e < a.k; e += L) {
        if (l.later[e] || l.cls[e] < 0) continue;
        double p = 0;
        for (int o = e; o < a.k; ++o) if (l.cls[o] == l.cls[e]) p += l.p[o];           // later ones are nobody else's to change
        l.p[e] = p;
        if (l.xmax > -INFINITY || l.x[e] != l.x[e]) {
            sl += exp2_32((l.x[e] - l.xmax) * a.c);
            if constexpr (TWO) sl1 += exp2_32((l.x[e] - l.xmax) * a.c1);
        }
    }
    const double s = group_sum<L>((double)sl), s1 = TWO ? group_sum<L>((double)sl1) : 0.0;
    wave_sync();
    for (int e = lane; e < a.k; e += L) if (l.later[e]) l.cls[e] = -1;
    if (lane == 0) { l.sl = s; l.sl1 = s1; }
    wave_sync();
}

// ---- bit map of the listed classes (listed_map.h) --------------------------------------------------------------------
template <typename T> __device__ __forceinline__ uint32_t vec_bits(const uint32_t* bits, int v) {
    const int b = BIT0 + v * ET<T>::VEC;
    const uint32_t byte = ((const uint8_t*)bits)[b >> 3];
    return ET<T>::IS_BF16 ? byte : (byte >> (b & 7)) & 15u;
}
// ---- loss and factors of a row from its sums -------------------------------------------------------------------------
// sr, s1: sums over the classes that are not listed, relative to their maximum m; S and the label's s1 over all of them,
// relative to the row's maximum.
struct RowSums { float xmax, m; double S, sr, a, s1, a1; };        // a, a1: 2^{(m - xmax) c}, 2^{(m - xmax) c1}
template <bool TWO, int K> __device__ __forceinline__ RowSums join_sums(const DistillArgs& a, const Listed<K>& l, float m, double sr, double s1) {
    RowSums s;
    const float both = fmaxf(m, l.xmax);
    s.xmax = both == -INFINITY ? 0.f : both;
    s.m = m == -INFINITY ? s.xmax : m;
    // a maximum of -inf: its sum is 0 (or NaN) and is taken as it is
    s.sr = sr;
    s.a = (double)exp2_32((s.m - s.xmax) * a.c);
    s.S = sr * s.a + (l.xmax == -INFINITY ? l.sl : l.sl * (double)exp2_32((l.xmax - s.xmax) * a.c));
    if constexpr (TWO) {
        s.a1 = (double)exp2_32((s.m - s.xmax) * a.c1);
        s.s1 = s1 * s.a1 + (l.xmax == -INFINITY ? l.sl1 : l.sl1 * (double)exp2_32((l.xmax - s.xmax) * a.c1));
    } else { s.a1 = s.a; s.s1 = s.S; }
    return s;
}
// A row of one wave or more: its numbers in scalar registers (next to 64 registers of scores others would be spilled).
template <int L> __device__ __forceinline__ float row_value(float v) {
    if constexpr (L == 64) return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); else return v;
}
template <int L> __device__ __forceinline__ double row_value(double v) { if constexpr (L == 64) return lane_value<64, 0>(v); else return v; }
template <int L> __device__ __forceinline__ RowSums row_value(const RowSums& s) {
    return {row_value<L>(s.xmax), row_value<L>(s.m), row_value<L>(s.S), row_value<L>(s.sr), row_value<L>(s.a), row_value<L>(s.s1), row_value<L>(s.a1)};
}
template <int L> __device__ __forceinline__ RowStats row_value(const RowStats& s) {
    return {row_value<L>(s.xl), row_value<L>(s.xr), row_value<L>(s.gl), row_value<L>(s.gr), row_value<L>(s.hl), row_value<L>(s.hr)};
}
// In every thread; the loss (three logarithms in 64 bits, a lane each) by one group.
__device__ __forceinline__ RowStats row_factors(const DistillArgs& a, const RowSums& s, bool hard, int flags, double pr) {
    const bool any = flags & 1, bad = flags & 2;
    RowStats st = {s.xmax, s.m, 0.f, 0.f, 0.f, 0.f};
    if (any) {
        const double f = (1.0 - a.w) * a.T, inv = 1.0 / s.S;
        st.gl = (float)(f * inv);
        st.gr = (float)(f * (s.a * inv - (pr > 0 && s.sr > 0 ? pr / s.sr : 0.0)));
    }
    if (hard) { const double h = a.w / s.s1; st.hl = (float)h; st.hr = (float)(h * s.a1); }
    if (bad || s.S != s.S || s.s1 != s.s1) st.gl = st.gr = st.hl = st.hr = NAN;
    if (!bad && ((!any && !hard) || s.S == 0)) st.xl = NAN;   // nothing to learn from, or no class to learn: zeros
    return st;
}
template <int L, int K> __device__ __forceinline__ double row_loss(const DistillArgs& a, const RowSums& s, const RowStats& st, bool hard, const Listed<K>& l, int lane, float xy) {
    double arg = s.s1;
    const double S = s.S, sr = s.sr;               // read in any case: a choice of members keeps the struct in memory
    if (lane == 0) arg = S;
    if (lane == 1) arg = sr;
    const double ln = ln_64(arg);
    const double lnS = lane_value<L, 0>(ln), lnr = lane_value<L, 1>(ln), ln1 = lane_value<L, 2>(ln);
    if (st.xl != st.xl) return 0.0;
    if (st.gl != st.gl) return NAN;
    double loss = 0;
    if (l.flags & 1) {
        // z = x / T; the sums are relative to xmax, that of the others to m, `cross` to the listed classes' largest score, whose
        // shares add up to 1 - p_r.  (Relative throughout: next to scores of 1e38 a log would vanish.)
        double kl = l.own - l.cross + lnS;
        if (l.xmax > -INFINITY) kl += (1.0 - l.pr) * (((double)s.xmax - (double)l.xmax) * (double)a.c * LN2);
        if (l.pr > 0) kl -= l.pr * (lnr + ((double)s.m - (double)s.xmax) * (double)a.c * LN2);
        loss = (1.0 - a.w) * a.T * a.T * kl;
    }
    if (hard) loss += a.w * (ln1 - ((double)xy - (double)s.xmax) * (double)a.c1 * LN2);
    return loss;
}

// The gradient of a score: of one side's classes, listed or not, relative to that side's reference.
template <typename T, bool TWO> struct Grad {
    float m, c, c1, g, h;
    __device__ __forceinline__ Grad(float m_, float c_, float c1_, float g_, float h_, float up) : m(m_), c(c_), c1(c1_), g((TWO ? g_ : g_ + h_) * up), h(h_ * up) {}
    __device__ __forceinline__ float operator()(float x) const {
        const float t = x - m, e = exp2_32(t * c);
        if constexpr (TWO) return fmaf(g, e, h * exp2_32(t * c1)); else return g * e;      // one temperature: h is in g
    }
};
template <typename T, bool TWO> __device__ __forceinline__ i32x4 grad_vec(const i32x4& v, const Grad<T, TWO>& g) {
    float f[ET<T>::VEC];
    unpack16<T>(v, f);
#pragma unroll
    for (int j = 0; j < ET<T>::VEC; ++j) f[j] = g(f[j]);
    return pack16<T>(f);
}

// One row by W waves, its scores held in registers (NV vectors a thread): read once, and with GRAD the gradient is
// written from there, so loss and gradient cost one read and one write of the scores.
// What the listed classes need is wave 0's.  The gradient is first written as if no class were listed; behind a barrier the
// listed ones and the label are written over.
// W = 1: a group of L lanes a row, L = 16 with at most 64 entries.
// The registers are cut for 4 waves a SIMD: 6 or 7 where they would do gave the same times, 8 spills (8192 x 65536 bf16: 454 us
// instead of 398).
template <typename T, int W, int L, int NV, bool TWO, bool GRAD>
__global__ __launch_bounds__(W == 1 ? 256 : W * 64, 4) void distill_row_kernel(DistillArgs a) {
    constexpr int VEC = ET<T>::VEC, G = W * L, ROWS = W == 1 ? 256 / L : 1, K = L == 64 ? MAX_K : 64, WORDS = (G * NV * VEC + 2 * BIT0 + 31) / 32;
    __shared__ uint32_t bits_[ROWS][WORDS];
    __shared__ Listed<K> l_[ROWS];
    __shared__ double rsum[2][W];
    __shared__ float rmax[W];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & (L - 1), tid = W == 1 ? lane : threadIdx.x, sub = W == 1 ? threadIdx.x / L : 0;
    const size_t r = (size_t)blockIdx.x * ROWS + sub;
    if (W == 1 && r >= (size_t)a.rows) return;
    const bool lead = W == 1 || wave == 0;
    uint32_t* bits = bits_[sub];
    Listed<K>& l = l_[sub];
    const int n = a.n;
    const T* x = (const T*)((const char*)a.x + r * a.stride * ET<T>::ES);
    const RowSpan<T> sp(x, n);

    const long long y = a.labels ? a.labels[r] : -1;
    const bool hard = a.w > 0.0 && y >= 0 && y < n;
    i32x4 v[NV];
    Entries<L, K> entries;
    if (lead) entries.load(a, r, lane);
    if (sp.nvec > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = load_vec(x, sp.vec_at(min(i * G + tid, sp.nvec - 1)));
    }
    float xe = tid < sp.edge ? load_score(x, sp.edge_at(tid)) : -INFINITY, xy = 0.f;
    if (lead) {
        listed_load<T>(a, entries, x, lane, l);
        if (hard) xy = load_score(x, (size_t)y);
    }
    for (int i = tid; i < WORDS; i += G) bits[i] = 0;
    group_sync<W>();
    if (lead) {
        bool dup = false;
        for (int e = lane; e < a.k; e += L)
            if (l.cls[e] >= 0) {
                const int b = BIT0 + l.cls[e] - sp.head;
                dup |= (atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31)) & 1;
            }
        if (lane == 0 && a.w > 0.0 && y >= n) l.flags |= 2;
        wave_sync();
        listed_sums<TWO, L>(a, lane, a.rest ? a.rest[r] : -INFINITY, l);
        if (group_any<L>(dup)) listed_merge<TWO, L>(a, lane, l);
    }
    group_sync<W>();

    // the maximum of the classes that are not listed; listed ones leave the registers
    float m = -INFINITY;
    if (xe > -INFINITY || xe != xe) {
        const int b = BIT0 + sp.edge_at(tid) - sp.head;
        if (bits[b >> 5] >> (b & 31) & 1) xe = -INFINITY;
        m = fmaxf(m, xe);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i * G + tid >= sp.nvec) v[i] = neg_inf_vec<T>();
        if (i * G < sp.nvec) {
            const uint32_t b = vec_bits<T>(bits, i * G + tid);
            if (b) drop_listed<T>(v[i], b);
            m = fmaxf(m, vec_max<T>(v[i]));
        }
    }
    m = group_max<L>(m);
    if constexpr (W > 1) {
        if (lane == 0) rmax[wave] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, rmax[w]);
    }

    // their sums
    const float ref = m == -INFINITY ? 0.f : m;
    float s = exp2_32((xe - ref) * a.c), s1 = TWO ? exp2_32((xe - ref) * a.c1) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i * G < sp.nvec) {
            float f[VEC];
            unpack16<T>(v[i], f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float t = f[j] - ref;
                s += exp2_32(t * a.c);
                if constexpr (TWO) s1 += exp2_32(t * a.c1);
            }
        }
    }
    double sr = group_sum<L>((double)s), sr1 = TWO ? group_sum<L>((double)s1) : 0.0;
    if constexpr (W > 1) {
        if (lane == 0) { rsum[0][wave] = sr; if constexpr (TWO) rsum[1][wave] = sr1; }
        __syncthreads();
        sr = sr1 = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) { sr += rsum[0][w]; if constexpr (TWO) sr1 += rsum[1][w]; }
    }
    const RowSums sum = row_value<L>(join_sums<TWO>(a, l, m, sr, sr1));
    const RowStats st = row_value<L>(row_factors(a, sum, hard, l.flags, l.pr));
    const bool empty = st.xl != st.xl;
    if (lead) {
        const double loss = row_loss<L>(a, sum, st, hard, l, lane, xy);
        if (lane == 0) {
            if (a.loss_rows) a.loss_rows[r] = loss; else a.loss[r] = (float)loss;
            a.stats[r] = st;
        }
    }
    if constexpr (!GRAD) {
        if (lead) for (int e = lane; e < a.k; e += L) a.probs[r * a.k + e] = l.cls[e] >= 0 ? (float)l.p[e] : -1.f;
    } else {
        T* dx = (T*)a.dx + r * (size_t)n;
        const Grad<T, TWO> g(st.xr, a.c, a.c1, st.gr, st.hr, a.scale);
        const bool same = (((uintptr_t)x ^ (uintptr_t)dx) & 15) == 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * G + tid < sp.nvec) {
                i32x4 o = grad_vec<T, TWO>(v[i], g);
                if (empty) o = zero16();
                const int at = sp.vec_at(i * G + tid);
                if (same) store_vec(dx, at, o);
                else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if constexpr (ET<T>::IS_BF16) ((uint16_t*)dx)[at + j] = (uint16_t)((uint32_t)o[j >> 1] >> (16 * (j & 1)));
                        else ((int*)dx)[at + j] = o[j];
                }
            }
        }
        if (tid < sp.edge) store_elem(dx, sp.edge_at(tid), empty ? 0.f : g(xe));
        group_sync<W>();
        if (lead && !empty) {
            const Grad<T, TWO> listed(st.xl, a.c, a.c1, st.gl, st.hl, a.scale);
            const float fp = a.fp * a.scale, w = a.w1 * a.scale;
            bool mine = false;
            for (int e = lane; e < a.k; e += L) {
                const int j = l.cls[e];
                if (j < 0) continue;
                float d = listed(l.x[e]) - fp * (float)l.p[e];
                if (hard && j == (int)y) { d -= w; mine = true; }
                store_elem(dx, j, d);
            }
            if (hard && !group_any<L>(mine) && lane == 0) store_elem(dx, (size_t)y, g(xy) - w);
        }
    }
}

// The loss alone, which needs no score twice: a row goes by in batches of four vectors a thread, with the next batch on its
// way, every thread with a running maximum and sums relative to it.  Bit map of SEG classes at a time.
template <typename T, int W, bool TWO>
__global__ __launch_bounds__(W * 64, W == 16 ? 4 : 6) void distill_stream_kernel(DistillArgs a) {
    constexpr int VEC = ET<T>::VEC, G = W * 64, NB = 4, BATCHES = SEG / VEC / (G * NB);
    __shared__ uint32_t bits[SEG_WORDS];
    __shared__ Listed<MAX_K> l;
    __shared__ double rsum[2][W];
    __shared__ float rmax[W];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, tid = threadIdx.x, n = a.n;
    const size_t r = blockIdx.x;
    const T* x = (const T*)((const char*)a.x + r * a.stride * ET<T>::ES);
    const RowSpan<T> sp(x, n);
    const bool lead = wave == 0;
    const long long y = a.labels ? a.labels[r] : -1;
    const bool hard = a.w > 0.0 && y >= 0 && y < n;
    float m = -INFINITY, s = 0.f, s1 = 0.f, xy = 0.f;
    // The sums of the segments before, relative to mf: 512 terms a thread of a segment, then at most eight segments, not one
    // chain of 4096.
    float mf = -INFINITY, sf = 0.f, s1f = 0.f;
    auto flush = [&] {
        if (mf != m) {                             // relative to -inf they are 0, or NaN
            if (mf > -INFINITY) {
                sf *= exp2_32((mf - m) * a.c);
                if constexpr (TWO) s1f *= exp2_32((mf - m) * a.c1);
            }
            mf = m;
        }
        sf += s; s = 0.f;
        if constexpr (TWO) { s1f += s1; s1 = 0.f; }
    };
    auto raise = [&](float to) {
        if (to > m) {
            s *= m == -INFINITY ? 0.f : exp2_32((m - to) * a.c);
            if constexpr (TWO) s1 *= m == -INFINITY ? 0.f : exp2_32((m - to) * a.c1);
            m = to;
        }
    };
    i32x4 nx[NB];
    auto load = [&](int v0) {
#pragma unroll
        for (int i = 0; i < NB; ++i) nx[i] = v0 + i * G + tid < sp.nvec ? load_vec(x, sp.vec_at(v0 + i * G + tid)) : neg_inf_vec<T>();
    };
    Entries<64, MAX_K> entries;
    if (lead) entries.load(a, r, lane);
    load(0);
    if (lead) {
        listed_load<T>(a, entries, x, lane, l);
        if (lane == 0 && a.w > 0.0 && y >= n) l.flags |= 2;
        wave_sync();
        listed_sums<TWO, 64>(a, lane, a.rest ? a.rest[r] : -INFINITY, l);
        if (hard) xy = load_score(x, (size_t)y);
    }
    const int some = segment_words(n);             // words of the bit map that are looked at
    for (int v0 = 0; v0 == 0 || v0 < sp.nvec; v0 += G * NB * BATCHES) {
        const int base = sp.vec_at(v0);            // the segment's first class; the row's ends go with the first segment
        __syncthreads();
        for (int i = tid; i < some; i += G) bits[i] = 0;
        __syncthreads();
        if (lead) {
            bool dup = false;
            for (int e = lane; e < a.k; e += 64) {
                const int j = l.cls[e], b = BIT0 + j - base;
                if (j >= base && j - base < SEG) dup |= (atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31)) & 1;
                dup |= j >= 0 && (j < base || j - base >= SEG);        // listed elsewhere: not seen by this bit map
            }
            if (v0 == 0 && group_any<64>(dup)) listed_merge<TWO, 64>(a, lane, l);
        }
        __syncthreads();
        if (v0 == 0 && tid < sp.edge) {
            const int j = sp.edge_at(tid);
            bool is_listed = false;
            for (int e = 0; e < a.k; ++e) is_listed |= l.cls[e] == j;
            if (!is_listed) {
                const float f = load_score(x, j);
                raise(f);
                const float t = f - (m == -INFINITY ? 0.f : m);
                s += exp2_32(t * a.c);
                if constexpr (TWO) s1 += exp2_32(t * a.c1);
            }
        }
#pragma unroll 1
        for (int b = 0; b < BATCHES && v0 + b * G * NB < sp.nvec; ++b) {
            i32x4 v[NB];
#pragma unroll
            for (int i = 0; i < NB; ++i) v[i] = nx[i];
            load(v0 + (b + 1) * G * NB);
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const uint32_t q = vec_bits<T>(bits, b * G * NB + i * G + tid);
                if (q) drop_listed<T>(v[i], q);
                top = fmaxf(top, vec_max<T>(v[i]));
            }
            raise(top);
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                float f[VEC];
                unpack16<T>(v[i], f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float t = f[j] - ref;
                    s += exp2_32(t * a.c);
                    if constexpr (TWO) s1 += exp2_32(t * a.c1);
                }
            }
        }
        flush();
    }
    const float all = block_reduce<W>(m, OpFMax(), rmax);
    const bool none = m == -INFINITY;              // then s is 0, or NaN
    const double sr = block_reduce<W>((double)sf * (none ? 1.0 : (double)exp2_32((m - all) * a.c)), OpSum(), rsum[0]);
    const double sr1 = TWO ? block_reduce<W>((double)s1f * (none ? 1.0 : (double)exp2_32((m - all) * a.c1)), OpSum(), rsum[1]) : 0.0;
    if (!lead) return;
    const RowSums sum = join_sums<TWO>(a, l, all, sr, sr1);
    const RowStats st = row_factors(a, sum, hard, l.flags, l.pr);
    const double loss = row_loss<64>(a, sum, st, hard, l, lane, xy);
    if (lane == 0) {
        if (a.loss_rows) a.loss_rows[r] = loss; else a.loss[r] = (float)loss;
        a.stats[r] = st;
    }
    for (int e = lane; e < a.k; e += 64) a.probs[r * a.k + e] = l.cls[e] >= 0 ? (float)l.p[e] : -1.f;
}

struct GradArgs {
    const void* x; size_t stride;
    const long long* idx; const long long* labels; const RowStats* stats; const float* probs;
    const float* g; int g_per_row; float scale; void* dx;
    int rows, n, k; float c, c1, fp, w;        // fp = (1 - w) T
};

// The gradient from a forward's factors.  W waves a piece of NV vectors a thread; blockIdx.x pieces of blockIdx.y-th rows
// (W = 1: four rows a workgroup, one piece each).  Written as if nothing were listed, the listed classes of the piece and
// the label over it.
template <typename T, int W, int NV, bool TWO>
__global__ __launch_bounds__(256) void distill_bwd_kernel(GradArgs a) {
    constexpr int VEC = ET<T>::VEC, G = W * 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, tid = W == 1 ? lane : threadIdx.x;
    const size_t r = W == 1 ? (size_t)blockIdx.x * 4 + wave : (size_t)blockIdx.y + (size_t)blockIdx.z * 65535;
    if (r >= (size_t)a.rows) return;
    const int n = a.n, v0 = W == 1 ? 0 : blockIdx.x * (G * NV);
    const T* x = (const T*)((const char*)a.x + r * a.stride * ET<T>::ES);
    T* dx = (T*)a.dx + r * (size_t)n;
    const RowSpan<T> sp(x, n);
    i32x4 v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) if (v0 + i * G + tid < sp.nvec) v[i] = load_vec(x, sp.vec_at(v0 + i * G + tid));
    const RowStats st = a.stats[r];
    const bool empty = st.xl != st.xl;
    const float up = (a.g ? a.g[a.g_per_row ? r : 0] : 1.f) * a.scale;
    const long long y = a.labels ? a.labels[r] : -1;
    const bool hard = a.w > 0.f && y >= 0 && y < n;
    const Grad<T, TWO> g(st.xr, a.c, a.c1, st.gr, st.hr, up), listed(st.xl, a.c, a.c1, st.gl, st.hl, up);
    const bool same = (((uintptr_t)x ^ (uintptr_t)dx) & 15) == 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (v0 + i * G + tid < sp.nvec) {
            i32x4 o = grad_vec<T, TWO>(v[i], g);
            if (empty) o = zero16();
            const int at = sp.vec_at(v0 + i * G + tid);
            if (same) store_vec(dx, at, o);
            else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if constexpr (ET<T>::IS_BF16) ((uint16_t*)dx)[at + j] = (uint16_t)((uint32_t)o[j >> 1] >> (16 * (j & 1)));
                    else ((int*)dx)[at + j] = o[j];
            }
        }
    }
    if (v0 == 0 && tid < sp.edge) { const int j = sp.edge_at(tid); store_elem(dx, j, empty ? 0.f : g(load_score(x, j))); }
    if (empty) return;
    group_sync<W>();
    // the classes of this piece; the row's edges belong to piece 0
    const int lo = sp.vec_at(v0), hi = min(lo + G * NV * VEC, sp.vec_at(sp.nvec));
    auto here = [&](long long j) { return (j >= lo && j < hi) || (v0 == 0 && (j < sp.head || j >= sp.vec_at(sp.nvec))); };
    bool mine = false;
    for (int e = tid; e < a.k; e += G) {
        const float p = a.probs[r * a.k + e];
        if (p < 0.f) continue;
        const long long j = a.idx[r * a.k + e];
        if (j < 0 || j >= n || !here(j)) continue;
        float d = listed(load_score(x, (size_t)j)) - a.fp * p * up;
        if (hard && j == y) { d -= a.w * up; mine = true; }
        store_elem(dx, (size_t)j, d);
    }
    if (!hard || !here(y)) return;
    if constexpr (W == 1) mine = __ballot(mine) != 0; else mine = __syncthreads_or(mine);
    if (tid == 0 && !mine) store_elem(dx, (size_t)y, g(load_score(x, (size_t)y)) - a.w * up);
}

// A gradient times what comes in, except the rows whose gradient is zero whatever that is (0 * inf would be NaN).
__global__ __launch_bounds__(256) void distill_scale_kernel(const float* dx, const RowStats* stats, const float* g, int g_per_row, unsigned n, unsigned total, float* out) {
    const unsigned i = blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const unsigned r = i / n;
    const float xl = stats[r].xl;
    out[i] = xl != xl ? 0.f : dx[i] * g[g_per_row ? r : 0];
}

// Sum of the rows' losses, added in row order within a thread and in a fixed order over them: the same bits every run.
// Eight loads are under way at a time (one after the other, 16384 rows took 5.5 us).
__global__ __launch_bounds__(1024) void loss_sum_kernel(const double* rows, int n, double scale, float* loss) {
    __shared__ double red[16];
    double s = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i - (int)threadIdx.x < n; i += 8 * 1024) {
        double v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = rows[min(i + j * 1024, n - 1)];
#pragma unroll
        for (int j = 0; j < 8; ++j) s += i + j * 1024 < n ? v[j] : 0.0;
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    s = wave_sum(threadIdx.x < 16 ? red[threadIdx.x] : 0.0);
    if (threadIdx.x == 0) *loss = (float)(s * scale);
}

bool bad_common(int dtype, const void* x, size_t stride, const void* idx, int rows, int ncls, int k, double T, double w) {
    return (dtype != STGCN_F32 && dtype != STGCN_BF16) || !x || !idx || rows < 1 || rows >= (1 << 24) || ncls < 1 || ncls > (1 << 20) || stride < (size_t)ncls
        || k < 1 || k > MAX_K || !temperature_ok(T) || !(w >= 0.0) || !(w <= 1.0);
}

// The widest row that fits in registers: 16 waves of 16 vectors a lane (64 registers of scores).
template <typename T> constexpr int row_fits() { return 1024 * 16 * ET<T>::VEC; }

template <typename T, bool TWO, bool GRAD> void launch_rows(const DistillArgs& a, hipStream_t s) {
    constexpr int VEC = ET<T>::VEC;
    const int nv = a.n / VEC;                      // at most, whatever the alignment
    const unsigned rows = (unsigned)a.rows, quads = (unsigned)((a.rows + 3) / 4), sixteens = (unsigned)((a.rows + 15) / 16);
    // As few waves a row as hold it in registers: what every row costs, some 1300 instructions of its first wave, then runs for
    // more rows at a time, and up to 64 entries four rows share a wave and its instructions.  Loss and gradient, us, by the
    // lanes (or waves) a row and vectors a lane, many rows of 256 MB (64 rows: all within 1 us of each other up to 8192 vectors):
    // 200000 x 128 float32 16 lanes x 2 81, x 8 86, a wave 260; 131072 x 512 16 lanes x 8 118, a wave x 4 196, four waves 491;
    // 65536 x 1024 a wave x 4 144, four x 4 264, x 8 280; 16384 x 4096 four x 4 115, x 8 110, eight 173; 8192 x 8192 four x 8
    // 105, eight x 8 117, x 16 154; 4096 x 16384 eight x 8 109, x 16 113, sixteen 209; 2048 x 32768 eight x 16 111, sixteen 155;
    // bf16 alike.  100 entries: 100000 x 240 float32 a wave x 2 158, x 4 152; 100000 x 500 a wave x 4 176, four waves 409.
    if (nv <= 32 && a.k <= 64) distill_row_kernel<T, 1, 16, 2, TWO, GRAD><<<sixteens, 256, 0, s>>>(a);
    else if (nv <= 128 && a.k <= 64) distill_row_kernel<T, 1, 16, 8, TWO, GRAD><<<sixteens, 256, 0, s>>>(a);
    else if (nv <= 256) distill_row_kernel<T, 1, 64, 4, TWO, GRAD><<<quads, 256, 0, s>>>(a);
    else if (nv <= 1024) distill_row_kernel<T, 4, 64, 4, TWO, GRAD><<<rows, 256, 0, s>>>(a);
    else if (nv <= 2048) distill_row_kernel<T, 4, 64, 8, TWO, GRAD><<<rows, 256, 0, s>>>(a);
    else if (nv <= 4096) distill_row_kernel<T, 8, 64, 8, TWO, GRAD><<<rows, 512, 0, s>>>(a);
    else if (nv <= 8192) distill_row_kernel<T, 8, 64, 16, TWO, GRAD><<<rows, 512, 0, s>>>(a);
    else distill_row_kernel<T, 16, 64, 16, TWO, GRAD><<<rows, 1024, 0, s>>>(a);
}
// The loss alone.  Wide rows go by in batches, by four waves a row, where there are two rows a compute unit or more; sixteen
// waves take few rows that no registers hold.  Row in registers / four waves / sixteen, us: 512 x 16384 float32 10.4 / 11.3 / 17,
// 1024 x 16384 21 / 17.5 / 36, 256 x 32768 10.7 / 12.9 / 11.3, 512 x 32768 20.8 / 16.8 / 23.9, 4096 x 65536 276 / 187 / 231,
// 512 x 32768 bf16 13.8 / 14.5 / 19.7, 1024 x 32768 27.7 / 22.1 / 41, 128 x 65536 13.3 / 15.4 / 13.9; with 8192 scores both
// first ones the same.
template <typename T, bool TWO> void launch_fwd(const DistillArgs& a, hipStream_t s) {
    if (a.n / ET<T>::VEC > 2048 && a.rows >= 512) distill_stream_kernel<T, 4, TWO><<<a.rows, 256, 0, s>>>(a);
    else if (a.n <= row_fits<T>()) launch_rows<T, TWO, false>(a, s);
    else distill_stream_kernel<T, 16, TWO><<<a.rows, 1024, 0, s>>>(a);
}
template <typename T, bool TWO> void launch_bwd(const GradArgs& a, hipStream_t s) {
    constexpr int VEC = ET<T>::VEC;
    const int nv = a.n / VEC > 0 ? a.n / VEC : 1;
    const unsigned quads = (unsigned)((a.rows + 3) / 4);
    // A wave a row with one or four vectors a lane, or a workgroup for 1024 vectors, us: 200000 x 60 float32 56 / 81 / 206,
    // 100000 x 240 39 / 46 / 102, 60000 x 400 - / 40 / 60, 30000 x 1000 - / 49 / 42.
    if (nv <= 64) distill_bwd_kernel<T, 1, 1, TWO><<<quads, 256, 0, s>>>(a);
    else if (nv <= 160) distill_bwd_kernel<T, 1, 4, TWO><<<quads, 256, 0, s>>>(a);
    else {
        const dim3 grid((nv + 1023) / 1024, a.rows < 65535 ? a.rows : 65535, (a.rows + 65534) / 65535);
        distill_bwd_kernel<T, 4, 4, TWO><<<grid, 256, 0, s>>>(a);
    }
}

DistillArgs fwd_args(const void* logits, size_t row_stride, const float* values, const int64_t* indices, const float* rest, const int64_t* labels,
                     int rows, int ncls, int k, double temperature, double label_weight) {
    return {logits, row_stride, values, (const long long*)indices, rest, label_weight > 0 ? (const long long*)labels : nullptr,
            nullptr, nullptr, nullptr, nullptr, nullptr, 1.f, rows, ncls, k, (float)(LOG2E / temperature), (float)LOG2E,
            (float)((1.0 - label_weight) * temperature), (float)label_weight, temperature, 1.0 / temperature, label_weight};
}
int loss_sum(const double* loss_rows, int rows, int reduction, float* loss, hipStream_t s) {
    if (reduction) loss_sum_kernel<<<1, 1024, 0, s>>>(loss_rows, rows, reduction == 1 ? 1.0 / rows : 1.0, loss);
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}

}  // namespace

extern "C" int stgcn_distill_fwd(int dtype, const void* logits, size_t row_stride, const float* values, const int64_t* indices,
                                 const float* rest, const int64_t* labels, int rows, int ncls, int k, double temperature,
                                 double label_weight, int reduction, float* loss, double* loss_rows, float* stats, float* probs, void* stream) {
    if (bad_common(dtype, logits, row_stride, indices, rows, ncls, k, temperature, label_weight) || !values || !loss || !stats || !probs
        || (label_weight > 0 && !labels) || reduction < 0 || reduction > 2 || (reduction && !loss_rows)) return STGCN_ERR_ARG;
    DistillArgs a = fwd_args(logits, row_stride, values, indices, rest, labels, rows, ncls, k, temperature, label_weight);
    a.loss_rows = reduction ? loss_rows : nullptr; a.loss = loss; a.stats = (RowStats*)stats; a.probs = probs;
    const bool two = label_weight > 0 && temperature != 1.0;
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == STGCN_BF16) { if (two) launch_fwd<bf16, true>(a, s); else launch_fwd<bf16, false>(a, s); }
    else { if (two) launch_fwd<float, true>(a, s); else launch_fwd<float, false>(a, s); }
    return loss_sum(loss_rows, rows, reduction, loss, (hipStream_t)stream);
}

extern "C" int stgcn_distill_bwd(int dtype, const void* logits, size_t row_stride, const int64_t* indices, const int64_t* labels,
                                 const float* stats, const float* probs, const float* grad, int grad_per_row, double scale, int rows,
                                 int ncls, int k, double temperature, double label_weight, void* dlogits, void* stream) {
    if (bad_common(dtype, logits, row_stride, indices, rows, ncls, k, temperature, label_weight) || !stats || !probs || !dlogits
        || (label_weight > 0 && !labels)) return STGCN_ERR_ARG;
    GradArgs a = {logits, row_stride, (const long long*)indices, label_weight > 0 ? (const long long*)labels : nullptr, (const RowStats*)stats,
                  probs, grad, grad_per_row, (float)scale, dlogits, rows, ncls, k, (float)(LOG2E / temperature), (float)LOG2E,
                  (float)((1.0 - label_weight) * temperature), (float)label_weight};
    const bool two = label_weight > 0 && temperature != 1.0;
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == STGCN_BF16) { if (two) launch_bwd<bf16, true>(a, s); else launch_bwd<bf16, false>(a, s); }
    else { if (two) launch_bwd<float, true>(a, s); else launch_bwd<float, false>(a, s); }
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}

extern "C" int stgcn_distill_scale(const float* dlogits, const float* stats, const float* grad, int grad_per_row, int rows, int ncls, float* out, void* stream) {
    if (!dlogits || !stats || !grad || !out || rows < 1 || ncls < 1 || (size_t)rows * (size_t)ncls >= (1u << 31)) return STGCN_ERR_ARG;
    const unsigned total = (unsigned)rows * (unsigned)ncls;
    distill_scale_kernel<<<(total + 255) / 256, 256, 0, (hipStream_t)stream>>>(dlogits, (const RowStats*)stats, grad, grad_per_row, (unsigned)ncls, total, out);
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}

extern "C" int stgcn_distill_step(int dtype, const void* logits, size_t row_stride, const float* values, const int64_t* indices,
                                  const float* rest, const int64_t* labels, int rows, int ncls, int k, double temperature,
                                  double label_weight, int reduction, float* loss, double* loss_rows, float* stats, float* probs, void* dlogits, void* stream) {
    if (bad_common(dtype, logits, row_stride, indices, rows, ncls, k, temperature, label_weight) || !values || !loss || !loss_rows || !stats
        || !probs || !dlogits || (label_weight > 0 && !labels) || reduction < 0 || reduction > 2) return STGCN_ERR_ARG;
    DistillArgs a = fwd_args(logits, row_stride, values, indices, rest, labels, rows, ncls, k, temperature, label_weight);
    a.loss_rows = reduction ? loss_rows : nullptr; a.loss = loss; a.dx = dlogits; a.scale = reduction == 1 ? (float)(1.0 / rows) : 1.f;
    a.stats = (RowStats*)stats; a.probs = probs;
    const bool two = label_weight > 0 && temperature != 1.0;
    const hipStream_t s = (hipStream_t)stream;
    if (ncls > (dtype == STGCN_BF16 ? row_fits<bf16>() : row_fits<float>())) {
        if (dtype == STGCN_BF16) { if (two) launch_fwd<bf16, true>(a, s); else launch_fwd<bf16, false>(a, s); }
        else { if (two) launch_fwd<float, true>(a, s); else launch_fwd<float, false>(a, s); }
        const int rc = stgcn_distill_bwd(dtype, logits, row_stride, indices, labels, stats, probs, nullptr, 0, reduction == 1 ? 1.0 / rows : 1.0, rows, ncls, k,
                                         temperature, label_weight, dlogits, stream);
        if (rc != STGCN_OK) return rc;
    } else if (dtype == STGCN_BF16) { if (two) launch_rows<bf16, true, true>(a, s); else launch_rows<bf16, false, true>(a, s); }
    else { if (two) launch_rows<float, true, true>(a, s); else launch_rows<float, false, true>(a, s); }
    return loss_sum(loss_rows, rows, reduction, loss, s);
}
