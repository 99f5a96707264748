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
// carries nearly all of the mass would leave nothing of the difference but rounding.
#include "scores.h"

namespace {

constexpr int MAX_K = 256;
constexpr int SEG = 65536;                    // classes per bit map (8 KB of LDS)
constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.6931471805599453094;

// What a row's forward leaves for its gradient: e^{z_j} = 2^{(x_j - xmax) c}, and the factors of the three sums.
struct RowStats { float xmax, gl, gr, g1; };   // gl = (1-w) T / S, gr = (1-w) T (1/S - p_r/S_r), g1 = w / sum e^x

struct DistillArgs {
    const void* x; size_t stride;
    const float* val; const long long* idx; const float* rest; const long long* labels;
    double* loss_rows; float* loss; RowStats* stats; float* probs;
    int n, k;
    float c, c1;                               // log2(e) / T, log2(e)
    double T, w;
};

// Running (maximum, sum of 2^{(x - maximum) c}, the same at temperature 1) of one thread's scores.
template <bool TWO> struct Online {
    float m = -INFINITY, s = 0.f, s1 = 0.f;
    __device__ __forceinline__ void raise(float to, float c, float c1) {
        if (to > m) {
            s *= m == -INFINITY ? 0.f : exp2_32((m - to) * c);
            if constexpr (TWO) s1 *= m == -INFINITY ? 0.f : exp2_32((m - to) * c1);
            m = to;
        }
    }
    __device__ __forceinline__ void add(float x, float c, float c1) {      // x <= m, or m = -inf and x = -inf
        if (x == -INFINITY) return;
        s += exp2_32((x - m) * c);
        if constexpr (TWO) s1 += exp2_32((x - m) * c1);
    }
};

template <typename T, bool TWO>
__global__ __launch_bounds__(256) void distill_fwd_kernel(DistillArgs a) {
    constexpr int VEC = ET<T>::VEC;
    __shared__ uint32_t bits[SEG / 32 + 1];
    __shared__ int li[MAX_K];
    __shared__ double redd[4];
    __shared__ float redf[4];
    const size_t r = blockIdx.x;
    const int tid = threadIdx.x, n = a.n, k = a.k;
    const T* x = (const T*)((const char*)a.x + r * a.stride * ET<T>::ES);

    // the teacher: thread q holds entry q
    int my = -1; bool bad = false; double tz = -INFINITY;
    if (tid < k) {
        const long long i = a.idx[r * k + tid];
        bad = i >= n;
        my = i < 0 || i >= n ? -1 : (int)i;
        if (my >= 0) {
            const float t = a.val[r * k + tid];
            bad = !(t < INFINITY);
            tz = bad ? -INFINITY : (double)t / a.T;
        }
        li[tid] = my;
    }
    const double rho = a.rest ? (double)a.rest[r] : -INFINITY;
    const bool soft = a.w < 1.0;
    const bool any = __syncthreads_or(my >= 0 && tz > -INFINITY) && soft;      // this row has a teacher
    const bool any_bad = __syncthreads_or(bad) || (any && !(rho < INFINITY));
    bool first = my >= 0;
    for (int q = 0; q < tid && q < k; ++q) if (li[q] == my) first = false;
    const double tmax = fmax(block_reduce<4>(tz, OpMax(), redd), any ? rho : -INFINITY);
    double A = 0, p = 0, pr = 0;
    if (any) {
        const double sum = block_reduce<4>(tid < k ? exp(tz - tmax) : 0.0, OpSum(), redd) + exp(rho - tmax);
        A = tmax + log(sum);
        p = exp(tz - A);
        pr = exp(rho - A);
    }
    long long y = -1;
    if constexpr (TWO) y = a.labels[r];
    else if (a.labels) y = a.labels[r];
    const bool hard = a.w > 0.0 && y >= 0;
    const bool bad_row = any_bad || (a.w > 0.0 && y >= n);

    // the student: a running maximum and sums over the classes that are not listed
    const float xl = first ? load_elem(x, my) : -INFINITY;
    Online<TWO> o;
    bool nan = xl != xl;
    const RowSpan<T> sp(x, n);
    for (int seg = 0; seg < n; seg += SEG) {
        __syncthreads();
        for (int i = tid; i < SEG / 32 + 1; i += 256) bits[i] = 0;
        __syncthreads();
        if (first && my >= seg && my < seg + SEG) atomicOr(&bits[(my - seg) >> 5], 1u << ((my - seg) & 31));
        __syncthreads();
        const int end = min(seg + SEG, n);
        for (int j = seg + tid; j < end; j += 256) {
            if (bits[(j - seg) >> 5] >> ((j - seg) & 31) & 1) continue;
            const float v = load_elem(x, j);
            nan |= v != v;
            o.raise(v, a.c, a.c1);
            o.add(v, a.c, a.c1);
        }
    }
    nan = __syncthreads_or(nan);
    const float xmax = block_reduce<4>(fmaxf(o.m, xl), OpFMax(), redf);
    double sr = 0, sl = 0, s1 = 0;
    if (o.m > -INFINITY) {
        sr = (double)o.s * (double)exp2_32((o.m - xmax) * a.c);
        if constexpr (TWO) s1 = (double)o.s1 * (double)exp2_32((o.m - xmax) * a.c1);
    }
    if (xl > -INFINITY) {
        sl = (double)exp2_32((xl - xmax) * a.c);
        if constexpr (TWO) s1 += (double)exp2_32((xl - xmax) * a.c1);
    }
    sr = block_reduce<4>(sr, OpSum(), redd);
    sl = block_reduce<4>(sl, OpSum(), redd);
    if constexpr (TWO) s1 = block_reduce<4>(s1, OpSum(), redd);
    const double S = sl + sr;
    if constexpr (!TWO) s1 = S;                            // temperature 1: one sum serves both terms
    double term = 0;
    if (any && p > 0) {
        const double lq = ((double)load_elem(x, my < 0 ? 0 : my) - (double)xmax) * (double)a.c * LN2 - log(S);
        if (my >= 0) term = p * (log(p) - lq);
    }
    double kl = block_reduce<4>(term, OpSum(), redd);
    // duplicates: the first occurrence carries the sum
    __shared__ double pk[MAX_K];
    if (tid < k) pk[tid] = my >= 0 ? p : 0.0;
    __syncthreads();
    if (tid < k && a.probs) {
        double t = 0;
        if (first) for (int q = tid; q < k; ++q) if (li[q] == my) t += pk[q];
        a.probs[r * k + tid] = first ? (float)t : -1.f;
    }
    if (tid == 0) {
        double loss = 0;
        RowStats st = {xmax, 0.f, 0.f, 0.f};
        if (any) {
            if (pr > 0) kl += pr * (log(pr) - log(sr) + log(S));
            loss += (1.0 - a.w) * a.T * a.T * kl;
            st.gl = (float)((1.0 - a.w) * a.T / S);
            st.gr = (float)((1.0 - a.w) * a.T * (1.0 / S - (pr > 0 && sr > 0 ? pr / sr : 0.0)));
        }
        if (hard && y < n) {
            loss += a.w * (log(s1) - ((double)load_elem(x, (size_t)y) - (double)xmax) * (double)a.c1 * LN2);
            st.g1 = (float)(a.w / s1);
        }
        const bool empty = (!any && !hard && !bad_row) || (xmax == -INFINITY && !nan && !bad_row);
        if (bad_row || nan) { loss = NAN; st.gl = st.gr = st.g1 = NAN; }
        if (empty) { loss = 0; st.xmax = NAN; }            // nothing to learn from, or no class to learn: zeros
        a.stats[r] = st;
        if (a.loss_rows) a.loss_rows[r] = loss;
        if (a.loss) a.loss[r] = (float)loss;
    }
}

struct GradArgs {
    const void* x; size_t stride;
    const long long* idx; const long long* labels; const RowStats* stats; const float* probs;
    const float* g; int g_per_row; float scale; void* dx;
    int n, k; float c, c1, fp, w;              // fp = (1 - w) T
};

template <typename T, bool TWO>
__global__ __launch_bounds__(256) void distill_bwd_kernel(GradArgs a) {
    const size_t r = blockIdx.x;
    const int tid = threadIdx.x, n = a.n, k = a.k;
    const T* x = (const T*)((const char*)a.x + r * a.stride * ET<T>::ES);
    T* dx = (T*)((char*)a.dx + r * (size_t)n * ET<T>::ES);
    const RowStats st = a.stats[r];
    const bool empty = st.xmax != st.xmax;
    const float g = (a.g ? a.g[a.g_per_row ? r : 0] : 1.f) * a.scale;
    const long long y = a.labels ? a.labels[r] : -1;
    auto grad = [&](float v, float gz) {
        const float t = v - st.xmax;
        const float e = exp2_32(t * a.c);
        return (TWO ? gz * e + st.g1 * exp2_32(t * a.c1) : (gz + st.g1) * e) * g;
    };
    for (int j = tid; j < n; j += 256) store_elem(dx, j, empty ? 0.f : grad(load_elem(x, j), st.gr));
    __syncthreads();
    if (empty) return;
    bool y_listed = false;
    if (tid < k) {
        const float p = a.probs[r * k + tid];
        if (p >= 0.f) {
            const long long j = a.idx[r * k + tid];
            float v = grad(load_elem(x, (size_t)j), st.gl) - a.fp * p * g;
            if (j == y && a.w > 0.f) { v -= a.w * g; y_listed = true; }
            store_elem(dx, (size_t)j, v);
        }
    }
    y_listed = __syncthreads_or(y_listed);
    if (tid == 0 && a.w > 0.f && y >= 0 && y < n && !y_listed)
        store_elem(dx, (size_t)y, grad(load_elem(x, (size_t)y), st.gr) - a.w * g);
}

// Sum of the rows' losses, added in row order within a thread and by fixed butterflies: the same bits every run.
__global__ __launch_bounds__(1024) void loss_sum_kernel(const double* rows, int n, double scale, float* loss) {
    __shared__ double red[16];
    double s = 0;
    for (int i = threadIdx.x; i < n; i += 1024) s += rows[i];
    s = block_reduce<16>(s, OpSum(), red);
    if (threadIdx.x == 0) *loss = (float)(s * scale);
}

bool bad_common(int dtype, const void* x, size_t stride, const void* idx, int rows, int ncls, int k, double T, double w) {
    return (dtype != STGCN_F32 && dtype != STGCN_BF16) || !x || !idx || rows < 1 || ncls < 1 || ncls > (1 << 20) || stride < (size_t)ncls
        || k < 1 || k > MAX_K || !(T > 0.0) || !(T < 1e30) || !(w >= 0.0) || !(w <= 1.0);
}

}  // namespace

extern "C" int stgcn_distill_fwd(int dtype, const void* logits, size_t row_stride, const float* values, const int64_t* indices,
                                 const float* rest, const int64_t* labels, int rows, int ncls, int k, double temperature,
                                 double label_weight, int reduction, float* loss, double* loss_rows, float* stats, float* probs, void* stream) {
    if (bad_common(dtype, logits, row_stride, indices, rows, ncls, k, temperature, label_weight) || !values || !loss || !stats || !probs
        || (label_weight > 0 && !labels) || reduction < 0 || reduction > 2 || (reduction && !loss_rows)) return STGCN_ERR_ARG;
    DistillArgs a = {logits, row_stride, values, (const long long*)indices, rest, label_weight > 0 ? (const long long*)labels : nullptr,
                     reduction ? loss_rows : nullptr, reduction ? nullptr : loss, (RowStats*)stats, probs, ncls, k,
                     (float)(LOG2E / temperature), (float)LOG2E, temperature, label_weight};
    const bool two = label_weight > 0 && temperature != 1.0;
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == STGCN_BF16) {
        if (two) distill_fwd_kernel<bf16, true><<<rows, 256, 0, s>>>(a); else distill_fwd_kernel<bf16, false><<<rows, 256, 0, s>>>(a);
    } else {
        if (two) distill_fwd_kernel<float, true><<<rows, 256, 0, s>>>(a); else distill_fwd_kernel<float, false><<<rows, 256, 0, s>>>(a);
    }
    if (reduction) loss_sum_kernel<<<1, 1024, 0, s>>>(loss_rows, rows, reduction == 1 ? 1.0 / rows : 1.0, loss);
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}

extern "C" int stgcn_distill_bwd(int dtype, const void* logits, size_t row_stride, const int64_t* indices, const int64_t* labels,
                                 const float* stats, const float* probs, const float* grad, int grad_per_row, double scale, int rows,
                                 int ncls, int k, double temperature, double label_weight, void* dlogits, void* stream) {
    if (bad_common(dtype, logits, row_stride, indices, rows, ncls, k, temperature, label_weight) || !stats || !probs || !dlogits
        || (label_weight > 0 && !labels)) return STGCN_ERR_ARG;
    GradArgs a = {logits, row_stride, (const long long*)indices, label_weight > 0 ? (const long long*)labels : nullptr, (const RowStats*)stats,
                  probs, grad, grad_per_row, (float)scale, dlogits, ncls, k, (float)(LOG2E / temperature), (float)LOG2E,
                  (float)((1.0 - label_weight) * temperature), (float)label_weight};
    const bool two = label_weight > 0 && temperature != 1.0;
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == STGCN_BF16) {
        if (two) distill_bwd_kernel<bf16, true><<<rows, 256, 0, s>>>(a); else distill_bwd_kernel<bf16, false><<<rows, 256, 0, s>>>(a);
    } else {
        if (two) distill_bwd_kernel<float, true><<<rows, 256, 0, s>>>(a); else distill_bwd_kernel<float, false><<<rows, 256, 0, s>>>(a);
    }
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}
