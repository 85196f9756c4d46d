// QuantizedLinear: Y = act(xs[m] ws[n] sum_k X[m,k] W[n,k] + b[n]) + R[m,n]; X and W in int8, both k-contiguous (W as a linear layer keeps it), Y, b
// and R in float32, float16 or bfloat16. The sums are int32 and exact (K below 2^17), everything behind them float32, rounded once. The reference has
// no such node: it runs MatMulInteger, a Cast, two Muls and the rest one after the other.
#include "mixed.h"
#include "gemm_tile.h"

#include <algorithm>

namespace mi355x {

struct QLinArgs {
    const int8_t* X; const int8_t* W; const float* xs; const float* ws;
    const void* bias; const void* residual; void* Y;
    int64_t M, N, K;
    int xs_step, ws_step;   // 0: one scale for all
    int activation;
    int64_t tiles_m, tiles_n;
};

// NaN stays NaN
template <int ACT>
__device__ __forceinline__ float activated(float v) {
    if (ACT == MI355X_ACT_RELU) return v < 0.0f ? 0.0f : v;
    if (ACT == MI355X_ACT_GELU) return gelu_erf(v);
    if (ACT == MI355X_ACT_SILU) return v / (1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
    return v;
}

// E results next to each other in row m, from column n on
template <class T, int ACT, int E>
__device__ __forceinline__ void qlin_store(const QLinArgs& p, int64_t m, int64_t n, const int (&acc)[E]) {
    if (m >= p.M || n >= p.N) return;
    const int64_t left = p.N - n;
    const float xs = p.xs[m * p.xs_step];
    float v[E], b[E], r[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = (float)acc[e] * xs * p.ws[p.ws_step ? (e < left ? n + e : n) : 0];
    if (p.bias) {
        load_values(b, static_cast<const T*>(p.bias) + n, left);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += b[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = activated<ACT>(v[e]);
    if (p.residual) {
        load_values(r, static_cast<const T*>(p.residual) + m * p.N + n, left);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += r[e];
    }
    store_values(static_cast<T*>(p.Y) + m * p.N + n, v, left);
}

// the 16 bytes from p on of which `left` belong to the row: the others as 0
__device__ __forceinline__ i32x4 row_bytes(const int8_t* p, int64_t left) {
    typedef i32x4 unaligned __attribute__((aligned(1)));
    if (left >= 16) return *reinterpret_cast<const unaligned*>(p);
    int8_t b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = i < left ? p[i] : (int8_t)0;
    return __builtin_bit_cast(i32x4, b);
}

// Any shape and alignment, operands straight from memory. A workgroup has 16 columns and 16 MT rows of Y, its eight waves take turns at the
// 128-byte lines of K and their sums meet in LDS.
template <class T, int ACT, int MT>
__global__ __launch_bounds__(512) void qlin_direct_kernel(QLinArgs p) {
    constexpr int WAVES = 8;
    __shared__ __attribute__((aligned(16))) i32x4 part[WAVES][MT][WAVE];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, l16 = lane % 16, lq = lane / 16;
    const int64_t n0 = (int64_t)blockIdx.x % p.tiles_n * 16, m0 = (int64_t)blockIdx.x / p.tiles_n * 16 * MT;
    const int8_t* w = p.W + std::min(n0 + l16, p.N - 1) * p.K;
    const int8_t* x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = p.X + std::min(m0 + 16 * t + l16, p.M - 1) * p.K;
    i32x4 acc[MT] = {};
    for (int64_t k = 128 * wave; k < p.K; k += 128 * WAVES) {
        i32x4 a[2], b[2][MT];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int64_t at = k + 64 * s + 16 * lq;
            a[s] = row_bytes(w + at, p.K - at);
#pragma unroll
            for (int t = 0; t < MT; ++t) b[s][t] = row_bytes(x[t] + at, p.K - at);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s], b[s][t], acc[t], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave >= MT) return;
    i32x4 sum = part[0][wave][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += part[w][wave][lane];
    const int s4[4] = {sum.x, sum.y, sum.z, sum.w};
    qlin_store<T, ACT, 4>(p, m0 + 16 * wave + l16, n0 + 4 * lq, s4);
}

template <class T, int ACT>
static void launch_qlin(QLinArgs p, hipStream_t st) {
    auto direct = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        p.tiles_n = ceil_div(p.N, (int64_t)16);
        p.tiles_m = ceil_div(p.M, (int64_t)(16 * MT));
        hipLaunchKernelGGL((qlin_direct_kernel<T, ACT, MT>), dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(512), 0, st, p);
    };
    if (p.M <= 16) direct(Int<1>{});
    else if (p.M <= 32) direct(Int<2>{});
    else direct(Int<4>{});
}

}  // namespace mi355x

extern "C" int mi355x_quantized_linear(const int8_t* X, const int8_t* W, const float* x_scale, const float* w_scale, const void* bias, const void* residual,
                                       void* Y, int64_t M, int64_t N, int64_t K, int64_t x_scale_count, int64_t w_scale_count, int activation, int type,
                                       void* stream) {
    using namespace mi355x;
    MI355X_REQUIRE(M >= 0 && N >= 0 && K >= 0, "quantized_linear: negative extent (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
    MI355X_REQUIRE(is_mixed_type(type), "quantized_linear: element type %d", type);
    MI355X_REQUIRE(activation >= MI355X_ACT_NONE && activation <= MI355X_ACT_SILU, "quantized_linear: activation %d", activation);
    MI355X_REQUIRE(K < (int64_t)1 << 17, "quantized_linear: K=%lld: sums of 2^17 products and more do not fit 32 bits", (long long)K);
    MI355X_REQUIRE(x_scale_count == 1 || x_scale_count == M, "quantized_linear: x_scale holds %lld values, expected 1 or M=%lld", (long long)x_scale_count, (long long)M);
    MI355X_REQUIRE(w_scale_count == 1 || w_scale_count == N, "quantized_linear: w_scale holds %lld values, expected 1 or N=%lld", (long long)w_scale_count, (long long)N);
    if (M == 0 || N == 0) return MI355X_OK;
    MI355X_REQUIRE((K == 0 || (X && W)) && x_scale && w_scale && Y, "quantized_linear: null pointer");
    MI355X_REQUIRE(M < (int64_t)1 << 31 && N < (int64_t)1 << 31 && grid_fits(ceil_div(M, (int64_t)16) * ceil_div(N, (int64_t)16), 512), "quantized_linear: too large");
    QLinArgs p = {X, W, x_scale, w_scale, bias, residual, Y, M, N, K, x_scale_count != 1, w_scale_count != 1, activation, 0, 0};
    with_type(type, [&](auto t) {
        using T = decltype(t);
        hipStream_t st = static_cast<hipStream_t>(stream);
        if (activation == MI355X_ACT_RELU) launch_qlin<T, MI355X_ACT_RELU>(p, st);
        else if (activation == MI355X_ACT_GELU) launch_qlin<T, MI355X_ACT_GELU>(p, st);
        else if (activation == MI355X_ACT_SILU) launch_qlin<T, MI355X_ACT_SILU>(p, st);
        else launch_qlin<T, MI355X_ACT_NONE>(p, st);
    });
    return check_launch("quantized_linear");
}
