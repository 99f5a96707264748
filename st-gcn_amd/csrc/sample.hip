// A label per row drawn from class scores with given random numbers.
//
// With w_j = e^{(x_j - max x) / T} and the classes in the order (score descending, class ascending):
//   keep the first top_k (0: all); of these the shortest prefix whose sum reaches top_p times the sum of all of these;
//   of these those with w_j >= min_p (the first class is always kept);
//   answer the first kept class j, by class number, with  sum_{i <= j, kept} w_i > u * sum of the kept w.
// All three cuts keep a prefix of that order, so the kept set is a pair (key, class): every class with a larger key, and
// of the classes with that key those up to that class.  Weights and sums are held in 64 bits: the answer is a whole number,
// and a sum in 32 bits would move it wherever u falls within 1e-7 of a border between two classes.
#include "scores.h"

namespace {

constexpr double LOG2E = 1.4426950408889634074;

struct SampleArgs {
    const void* x; size_t stride; const float* u;
    const float* tp; const int* kp; const float* pp; const float* qp;      // per row, or null: the scalars
    float t; int k; float p, q;
    long long* labels; float* logp; int n;
};

constexpr int W = 16, NT = W * 64;

template <typename T>
__global__ __launch_bounds__(NT) void sample_kernel(SampleArgs a) {
    __shared__ unsigned long long redu[W];
    __shared__ int redi[W];
    __shared__ double redd[W];
    const size_t r = blockIdx.x;
    const int tid = threadIdx.x, n = a.n;
    const T* x = (const T*)((const char*)a.x + r * a.stride * ET<T>::ES);
    const float u = a.u[r], t = a.tp ? a.tp[r] : a.t, p = a.pp ? a.pp[r] : a.p, q = a.qp ? a.qp[r] : a.q;
    int k = a.kp ? a.kp[r] : a.k;
    auto answer = [&](int label, float lp) { if (tid == 0) { a.labels[r] = label; a.logp[r] = lp; } };

    unsigned long long best = 0;
    for (int j = tid; j < n; j += NT) {
        const unsigned long long v = ((unsigned long long)score_key(load_elem(x, j)) << 32) | (uint32_t)~j;
        if (v > best) best = v;
    }
    best = block_reduce<W>(best, OpMax(), redu);
    const uint32_t top = (uint32_t)(best >> 32);
    if (top == KEY_NAN || !(t >= 0.f) || !(t < INFINITY) || k < 0 || !(p > 0.f) || !(p <= 1.f) || !(q >= 0.f) || !(q <= 1.f) || !(u >= 0.f) || !(u < 1.f))
        return answer(-1, NAN);
    if (top == KEY_NEG_INF) return answer(-1, -INFINITY);
    if (t == 0.f || k == 1) return answer((int)~(uint32_t)best, 0.f);
    if (k == 0 || k > n) k = n;
    const float xmax = key_score(top);
    const double c = LOG2E / (double)t;
    auto weight = [&](float v) { return v == xmax ? 1.0 : exp2_64(((double)v - (double)xmax) * c); };

    uint32_t tk = 0; int ti = n;                           // kept: key > tk, or key == tk and class <= ti
    auto kept = [&](uint32_t key, int j) { return key > tk || (key == tk && j <= ti); };
    auto count = [&](auto pred) {
        int m = 0;
        for (int j = tid; j < n; j += NT) m += pred(score_key(load_elem(x, j)), j) ? 1 : 0;
        return block_reduce<W>(m, OpSum(), redi);
    };
    auto mass = [&](auto pred) {
        double m = 0;
        for (int j = tid; j < n; j += NT) { const float v = load_elem(x, j); if (pred(score_key(v), j)) m += weight(v); }
        return block_reduce<W>(m, OpSum(), redd);
    };
    // the largest key v with enough(v), which holds for 0 and not beyond `top`
    auto bisect = [&](auto enough) {
        uint32_t lo = tk, hi = top;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            if (enough(mid)) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    // the class of the m-th one with key v (among the kept)
    auto nth = [&](uint32_t v, int m) {
        int lo = 0, hi = n - 1;
        while (lo < hi) {
            const int mid = lo + (hi - lo) / 2;
            if (count([&](uint32_t key, int j) { return key == v && j <= mid; }) >= m) hi = mid; else lo = mid + 1;
        }
        return lo;
    };
    if (k < n) {
        const uint32_t v = bisect([&](uint32_t mid) { return count([&](uint32_t key, int) { return key >= mid; }) >= k; });
        const int above = count([&](uint32_t key, int) { return key > v; });
        ti = nth(v, k - above);
        tk = v;
    }
    if (p < 1.f) {
        const double target = (double)p * mass(kept);
        const uint32_t v = bisect([&](uint32_t mid) { return mass([&](uint32_t key, int j) { return kept(key, j) && key >= mid; }) >= target; });
        const double above = mass([&](uint32_t key, int) { return key > v; }), one = weight(key_score(v));
        const int ties = count([&](uint32_t key, int j) { return key == v && kept(key, j); });
        int m = ties;
        if (above + (ties - 1) * one >= target) {          // not all of them: the smallest m with above + m * one >= target
            m = (int)ceil((target - above) / one);
            if (m < 1) m = 1;
            if (m > ties) m = ties;
            while (m > 1 && above + (m - 1) * one >= target) --m;
            while (m < ties && above + m * one < target) ++m;
        }
        ti = nth(v, m);
        tk = v;
    }
    if (q > 0.f) {
        uint32_t lo = tk, hi = top;                        // the smallest key that weighs enough
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (weight(key_score(mid)) >= (double)q) hi = mid; else lo = mid + 1;
        }
        if (lo > tk) { tk = lo; ti = n; }
    }
    const double total = mass(kept), target = (double)u * total;
    double before = 0;
    __shared__ int found; __shared__ double wave_sum[W];
    int last = 0;
    for (int base = 0; base < n; base += NT) {
        const int j = base + tid;
        double w = 0;
        if (j < n) { const float v = load_elem(x, j); if (kept(score_key(v), j)) w = weight(v); }
        double s = w;                                      // inclusive prefix within the wave
        for (int d = 1; d < 64; d <<= 1) { const double o = __shfl_up(s, d); if ((tid & 63) >= d) s += o; }
        __syncthreads();
        if (tid == 0) found = n;
        if ((tid & 63) == 63) wave_sum[tid >> 6] = s;
        __syncthreads();
        double b = before;
        for (int i = 0; i < (tid >> 6); ++i) b += wave_sum[i];
        if (w > 0 && b + s > target) atomicMin(&found, j);
        for (int i = 0; i < W; ++i) before += wave_sum[i];
        __syncthreads();
        if (found < n) break;
        const unsigned long long any = w > 0 ? (unsigned long long)j + 1 : 0;
        last = max(last, (int)block_reduce<W>(any, OpMax(), redu));
    }
    const int j = found < n ? found : last - 1;            // u next to 1 and the last sum rounded down
    answer(j, (float)log(weight(load_elem(x, j)) / total));
}

}  // namespace

extern "C" int stgcn_sample_labels(int dtype, const void* logits, size_t row_stride, const float* u, const float* temperatures, float temperature,
                                   const int* top_ks, int top_k, const float* top_ps, float top_p, const float* min_ps, float min_p,
                                   int64_t* labels, float* logp, int rows, int ncls, void* stream) {
    if (!logits || !u || !labels || !logp || rows < 1 || ncls < 1 || ncls > (1 << 20) || row_stride < (size_t)ncls) return STGCN_ERR_ARG;
    SampleArgs a = {logits, row_stride, u, temperatures, top_ks, top_ps, min_ps, temperature, top_k, top_p, min_p, (long long*)labels, logp, ncls};
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == STGCN_BF16) sample_kernel<bf16><<<rows, NT, 0, s>>>(a);
    else if (dtype == STGCN_F32) sample_kernel<float><<<rows, NT, 0, s>>>(a);
    else return STGCN_ERR_ARG;
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}
