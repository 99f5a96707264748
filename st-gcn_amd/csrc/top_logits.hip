// The largest k scores of every row, with their classes, and the log of what the other classes weigh together.
//
// Classes are ordered by (score descending, class ascending); NaN comes first.  rest = log sum over the unlisted
// classes of e^{x/T}, summed over them alone (never as a difference of sums).
#include "scores.h"

namespace {

constexpr int MAX_K = 256;
constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.6931471805599453094;

// position in the order as one number: larger is earlier
__device__ __forceinline__ unsigned long long place(uint32_t key, int j) { return ((unsigned long long)key << 32) | (uint32_t)~j; }

// One workgroup per row, the k largest one after the other.
template <typename T>
__global__ __launch_bounds__(256) void top_logits_kernel(const T* logits, size_t stride, int n, int k, float c, double T_, float* values,
                                                         long long* indices, float* rest) {
    __shared__ unsigned long long red[4];
    __shared__ float redf[4];
    __shared__ double redd[4];
    const size_t r = blockIdx.x;
    const T* x = (const T*)((const char*)logits + r * stride * ET<T>::ES);
    unsigned long long last = ~0ull;
    for (int q = 0; q < k; ++q) {
        unsigned long long best = 0;
        for (int j = threadIdx.x; j < n; j += 256) {
            const unsigned long long p = place(score_key(load_elem(x, j)), j);
            if (p > best && (q == 0 || p < last)) best = p;
        }
        last = block_reduce<4>(best, OpMax(), red);
        if (threadIdx.x == 0) {
            const int j = (int)~(uint32_t)last;
            values[r * k + q] = load_elem(x, j);
            indices[r * k + q] = j;
        }
    }
    float m = -INFINITY, s = 0.f;
    bool nan = false;
    for (int j = threadIdx.x; j < n; j += 256) {
        const float v = load_elem(x, j);
        if (place(score_key(v), j) < last) { m = fmaxf(m, v); nan |= v != v; }
    }
    nan = __syncthreads_or(nan);
    m = block_reduce<4>(m, OpFMax(), redf);
    for (int j = threadIdx.x; j < n; j += 256) {
        const float v = load_elem(x, j);
        if (place(score_key(v), j) < last && v > -INFINITY) s += v == m ? 1.f : exp2_32((v - m) * c);
    }
    const double sum = block_reduce<4>((double)s, OpSum(), redd);
    if (threadIdx.x == 0) rest[r] = nan ? NAN : m == -INFINITY ? -INFINITY : (float)((double)m / T_ + log(sum));
}

}  // namespace

extern "C" int stgcn_top_logits(int dtype, const void* logits, size_t row_stride, int rows, int ncls, int k, double temperature,
                                float* values, int64_t* indices, float* rest, void* stream) {
    if (!logits || !values || !indices || !rest || rows < 1 || ncls < 1 || ncls > (1 << 20) || row_stride < (size_t)ncls || k < 1 || k > MAX_K
        || k > ncls || !(temperature > 0.0) || !(temperature < 1e30)) return STGCN_ERR_ARG;
    const float c = (float)(LOG2E / temperature);
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == STGCN_BF16) top_logits_kernel<bf16><<<rows, 256, 0, s>>>((const bf16*)logits, row_stride, ncls, k, c, temperature, values, (long long*)indices, rest);
    else if (dtype == STGCN_F32) top_logits_kernel<float><<<rows, 256, 0, s>>>((const float*)logits, row_stride, ncls, k, c, temperature, values, (long long*)indices, rest);
    else return STGCN_ERR_ARG;
    return hipGetLastError() == hipSuccess ? STGCN_OK : STGCN_ERR_LAUNCH;
}
