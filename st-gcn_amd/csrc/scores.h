// Device helpers shared by the kernels over class scores (top_logits, distill, sample).
//
// A row of scores is [ncls] float32 or bf16, contiguous, at any element alignment: a row of an odd class count starts
// anywhere.  RowSpan splits it into the elements in front of the first 16-byte boundary, whole 16-byte vectors, and the
// elements behind the last one, so that no load or store touches a byte outside the row.
#pragma once
#include "stgcn_common.h"

// Temperatures T whose log2(e) / T is a float32 number, with room: below, 0 * inf would make NaN of a row's largest score.
inline bool temperature_ok(double T) { return T > 1e-30 && T < 1e30; }

template <typename T> struct RowSpan {
    static constexpr int VEC = ET<T>::VEC;
    int head, nvec, edge;                  // elements in front, vectors, elements in front and behind together
    __device__ __forceinline__ RowSpan(const void* row, int n) {
        const int off = (int)((uintptr_t)row & 15) / ET<T>::ES;
        head = off ? VEC - off : 0;
        if (head > n) head = n;
        nvec = (n - head) / VEC;
        edge = n - nvec * VEC;
    }
    __device__ __forceinline__ int vec_at(int v) const { return head + v * VEC; }           // first class of vector v
    __device__ __forceinline__ int edge_at(int e) const { return e < head ? e : e + nvec * VEC; }   // class of edge element e
};

// Named as global memory: a pointer that went through a struct is a flat one to the compiler, and flat loads are waited
// for with the LDS.
#define STGCN_GLOBAL __attribute__((address_space(1)))
template <typename T> __device__ __forceinline__ i32x4 load_vec(const T* row, int at) {
    return *(const STGCN_GLOBAL i32x4*)((uintptr_t)row + (size_t)at * ET<T>::ES);
}
template <typename T> __device__ __forceinline__ void store_vec(T* row, int at, const i32x4& raw) {
    *(STGCN_GLOBAL i32x4*)((uintptr_t)row + (size_t)at * ET<T>::ES) = raw;
}
template <typename T> __device__ __forceinline__ float load_score(const T* row, size_t at) {
    if constexpr (ET<T>::IS_BF16) return bf16_bits_to_f32(*(const STGCN_GLOBAL uint16_t*)((uintptr_t)row + at * 2));
    else return *(const STGCN_GLOBAL float*)((uintptr_t)row + at * 4);
}

__device__ __forceinline__ int lanes_below(unsigned long long mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// the elements of a vector whose bit is set become -inf
template <typename T> __device__ __forceinline__ void drop_listed(i32x4& v, uint32_t b) {
    if constexpr (ET<T>::IS_BF16) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t w = (uint32_t)v[q];
            if (b >> (2 * q) & 1) w = (w & 0xFFFF0000u) | 0xFF80u;
            if (b >> (2 * q + 1) & 1) w = (w & 0xFFFFu) | 0xFF800000u;
            v[q] = (int)w;
        }
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) if (b >> q & 1) v[q] = (int)0xFF800000u;
    }
}
template <typename T> __device__ __forceinline__ i32x4 neg_inf_vec() {
    const int w = ET<T>::IS_BF16 ? (int)0xFF80FF80u : (int)0xFF800000u;
    i32x4 v = {w, w, w, w};
    return v;
}
template <typename T> __device__ __forceinline__ float vec_max(const i32x4& v) {
    float f[ET<T>::VEC];
    unpack16<T>(v, f);
    float m = f[0];
#pragma unroll
    for (int j = 1; j < ET<T>::VEC; ++j) m = fmaxf(m, f[j]);
    return m;
}

// Order of the scores as unsigned integers: a > b as floats <=> key(a) > key(b); -0 and 0 are one key; NaN is above
// everything.
constexpr uint32_t KEY_NAN = 0xFFFFFFFFu, KEY_NEG_INF = 0x007FFFFFu;
__device__ __forceinline__ uint32_t score_key(float x) {
    if (x != x) return KEY_NAN;
    const uint32_t b = __float_as_uint(x + 0.f);           // -0 + 0 = 0
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_score(uint32_t k) {
    if (k == KEY_NAN) return __uint_as_float(0x7FC00000u);
    return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu));
}

// v_exp_f32: 2^y to one unit in the last place, 0 below 2^-126.
__device__ __forceinline__ float exp2_32(float y) { return __builtin_amdgcn_exp2f(y); }

// 2^y in 64 bits for y <= 1000: y = n + f, |f| <= 1/2, and 2^f = 1 + f q(f), q the polynomial of degree 8 that agrees with
// (2^f - 1) / f at the nine Chebyshev points of [-1/2, 1/2] (3.7e-14 of the value at most, exactly 1 at y = 0).  Every
// 64-bit operation here, roundings and ldexp among them, issues at the rate of an add (4.8 cycles a wave and SIMD
// measured, v_exp_f32 10.8).  N values at once: their chains side by side hide the latency.
template <int N> __device__ __forceinline__ void exp2_64(const double* y, double* out) {
    double f[N], p[N];
    int n[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const double v = fmax(y[e], -1100.0), r = rint(v);
        f[e] = v - r;
        n[e] = (int)r;
        p[e] = 1.0203121063391729e-07;
    }
    constexpr double Q[9] = {1.3255224878668817e-06, 1.525268684626772e-05, 0.00015403455852453838, 0.0013333558179043112, 0.009618129159402558,
                             0.055504108664760424, 0.2402265069581299, 0.6931471805599453, 1.0};
#pragma unroll
    for (int q = 0; q < 9; ++q) {
        double c = Q[q];
        asm volatile("" : "+s"(c));               // in scalar registers, here: else all are carried along, in 20 vector registers
#pragma unroll
        for (int e = 0; e < N; ++e) p[e] = fma(p[e], f[e], c);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = ldexp(p[e], n[e]);
}
__device__ __forceinline__ double exp2_64(double y) {
    double w;
    exp2_64<1>(&y, &w);
    return w;
}

// ln x in 64 bits: x = m 2^e, y = v_log_f32(m), and one Newton step on 2^y = m: y + (m 2^-y - 1) log2(e), within 1e-14.
// 0 and +inf answer -inf and +inf, less than 0 and NaN answer NaN.
__device__ __forceinline__ double ln_64(double x) {
    int e;
    const double m = frexp(x, &e);
    if (!(m > 0) || m == INFINITY) return m == 0 ? -INFINITY : m == INFINITY ? m : NAN;
    const double y = (double)__builtin_amdgcn_logf((float)m);
    return ((double)e + y + fma(m, exp2_64(-y), -1.0) * 1.4426950408889634074) * 0.6931471805599453094;
}

// ---- reductions of a workgroup of W waves: every thread gets the result; `red` is W entries of LDS -------------------
struct OpMax { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; } };
struct OpFMax { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct OpSum { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; } };

template <typename V, typename Op> __device__ __forceinline__ V wave_reduce(V v, Op op) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = op(v, __shfl_xor(v, d));
    return v;
}
// Sum over the wave by adds through the data-parallel crossbar (rows of 16 by shifts, then row to row), for every lane.
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_add(double v) {
    const long long b = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROWS, 0xF, true), hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xF, true);
    return v + __longlong_as_double((long long)hi << 32 | (uint32_t)lo);
}
__device__ __forceinline__ double wave_sum(double v) {
    v = dpp_add<0x111, 0xF>(v);                            // row_shr 1, 2, 4, 8: lane 15 of a row holds the row's sum
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);                            // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
    v = dpp_add<0x143, 0xC>(v);
    const long long b = __double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)b, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), 63);
    return __longlong_as_double((long long)hi << 32 | lo);
}

// Maximum over the wave the same way (fmaxf: NaN is no number).
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_max(float v) {
    const int o = __builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, ROWS, 0xF, false);    // itself where there is none
    return fmaxf(v, __int_as_float(o));
}
__device__ __forceinline__ float wave_max(float v) {
    v = dpp_max<0x111, 0xF>(v);
    v = dpp_max<0x112, 0xF>(v);
    v = dpp_max<0x114, 0xF>(v);
    v = dpp_max<0x118, 0xF>(v);
    v = dpp_max<0x142, 0xA>(v);
    v = dpp_max<0x143, 0xC>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// The same for 64-bit integers.
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned long long dpp_add(unsigned long long v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, true);
    return v + ((unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ unsigned long long wave_sum(unsigned long long v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    v = dpp_add<0x143, 0xC>(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63);
    return (unsigned long long)hi << 32 | lo;
}

template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true); }
// The sum over this lane and those below it: the same steps, before the last lane's is handed to all.
template <typename V> __device__ __forceinline__ V wave_scan(V v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    return dpp_add<0x143, 0xC>(v);
}
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, ROWS, 0xF, false);
    return o > v ? o : v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = dpp_max<0x111, 0xF>(v);
    v = dpp_max<0x112, 0xF>(v);
    v = dpp_max<0x114, 0xF>(v);
    v = dpp_max<0x118, 0xF>(v);
    v = dpp_max<0x142, 0xA>(v);
    v = dpp_max<0x143, 0xC>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Groups of L lanes: a whole wave (64), or a row of 16 (four groups side by side, for which one instruction serves all four).
// Lane WHO's value for every lane of its group.
template <int L, int WHO> __device__ __forceinline__ int lane_value(int v) {
    if constexpr (L == 64) return __builtin_amdgcn_readlane(v, WHO);
    else return __builtin_amdgcn_update_dpp(0, v, 0x150 + WHO, 0xF, 0xF, true);          // row_newbcast
}
template <int L, int WHO> __device__ __forceinline__ double lane_value(double v) {
    const long long b = __double_as_longlong(v);
    const uint32_t lo = (uint32_t)lane_value<L, WHO>((int)b), hi = (uint32_t)lane_value<L, WHO>((int)(b >> 32));
    return __longlong_as_double((long long)hi << 32 | lo);
}
template <int L> __device__ __forceinline__ double group_sum(double v) {
    if constexpr (L == 64) return wave_sum(v);
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    return lane_value<16, 15>(v);
}
template <int L> __device__ __forceinline__ float group_max(float v) {
    if constexpr (L == 64) return wave_max(v);
    v = dpp_max<0x111, 0xF>(v);
    v = dpp_max<0x112, 0xF>(v);
    v = dpp_max<0x114, 0xF>(v);
    v = dpp_max<0x118, 0xF>(v);
    return __int_as_float(lane_value<16, 15>(__float_as_int(v)));
}
template <int L> __device__ __forceinline__ bool group_any(bool b) {
    const unsigned long long m = __ballot(b);
    if constexpr (L == 64) return m != 0;
    return (m >> (threadIdx.x & 48) & 0xFFFF) != 0;
}

template <int W, typename V, typename Op> __device__ __forceinline__ V block_reduce(V v, Op op, V* red) {
    v = wave_reduce(v, op);
    if constexpr (W == 1) return v;
    __syncthreads();                                       // the previous use of `red` has been read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    V r = red[0];
#pragma unroll
    for (int w = 1; w < W; ++w) r = op(r, red[w]);
    return r;
}
