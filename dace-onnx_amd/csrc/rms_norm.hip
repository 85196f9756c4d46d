// SkipRMSNormalization: s = x + skip, y = s / sqrt(mean(s^2) + eps) * gain, and y in eight bits: q = round(y / scale) with scale = max |y| / 127 of
// the row, halves to even. Arrays in float32, float16 or bfloat16; everything between the loads and the stores in float32, y from the sum as it is
// before it is rounded for the caller. The reference has no such node.
//
// One pass over memory: a row stays in registers from its load to its last store. Per row the threads sum the squares, then take the largest
// |y|; both are exchanged in the wave by DPP and between waves through LDS.
//   rms_norm_rows<T, TH, NV>  TH threads to a row, NV vectors of 16 bytes to a thread: a wave while two vectors to a lane hold the row, then 256 threads, whose loads are in
//                             flight together, then 1024, so that no thread holds more than 32 values and their residuals
//   rms_norm_long             longer rows: one workgroup sweeps them three times, element by element: 1024 x 40000 in float32 240 us, 0.49 GB at 2 TB/s
// Bound by the bytes: 16384 x 4096 in bfloat16 with residual, sum and eight bits 84 us, 5.6 TB/s (a copy of 1 GiB 5.1); 1777 x 1001 in float32 7.1 us. Few rows by the
// launch and three trips (memory, two exchanges): 4 x 2048 3.2 us, of which an empty launch is 1.6. Rows at any address: 16-byte accesses wherever they lie. Narrow rows leave lanes
// idle: 128 values in bfloat16, a norm of each head, are 16 vectors for the 64 lanes of a wave: 65536 of them 20 us, 1.7 TB/s.
#include "mixed.h"

namespace mi355x {

struct RmsArgs {
    const void* X; const void* skip; const void* gain;
    void* Y; void* Sum; int8_t* Q; float* q_scale;
    int64_t rows, cols;
    float eps;
};

__device__ __forceinline__ uint32_t row16_max_u32(uint32_t v) {
    auto step = [&](auto control) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(control)::value, 0xf, 0xf, false);
        v = v > o ? v : o;
    };
    step(Int<DPP_QUAD_XOR1>{});
    step(Int<DPP_QUAD_XOR2>{});
    step(Int<DPP_ROW_HALF_MIRROR>{});
    step(Int<DPP_ROW_MIRROR>{});
    return v;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = row16_max_u32(v);
    uint32_t m = 0;
#pragma unroll
    for (int lane = 0; lane < WAVE; lane += 16) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
        m = m > o ? m : o;
    }
    return m;
}

// of TH threads, a multiple of 64; `part` has room for a value of each of the workgroup's waves and is free again at the next barrier but one
template <int TH>
__device__ __forceinline__ float threads_sum(float v, float* part) {
    v = wave_sum(v);
    if constexpr (TH > WAVE) {
        const int wave = threadIdx.x / WAVE, first = wave - wave % (TH / WAVE);
        part[wave] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < TH / WAVE; ++w) v += part[first + w];
    }
    return v;
}
template <int TH>
__device__ __forceinline__ uint32_t threads_max(uint32_t v, uint32_t* part) {
    v = wave_max_u32(v);
    if constexpr (TH > WAVE) {
        const int wave = threadIdx.x / WAVE, first = wave - wave % (TH / WAVE);
        part[wave] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < TH / WAVE; ++w) v = v > part[first + w] ? v : part[first + w];
    }
    return v;
}

// What the squares are taken of: squares of values from 2^64 on do not fit float32, those below 2^-63 are lost. Where that matters the row is
// summed again, scaled by a power of two: 2^31 squares of the largest values times 2^-96 stay below 2^96, those of rows whose mean square is below 2^-80
// times 2^88 below 2^127, and the least value above zero is then 2^-61.
constexpr float RMS_UP = 0x1p88f, RMS_DOWN = 0x1p-96f;
__device__ __forceinline__ float rms_rescale(float mean_square, float eps) {
    if (mean_square == __builtin_inff()) return RMS_DOWN;
    return mean_square < 0x1p-80f && eps < 0x1p-60f ? RMS_UP : 1.0f;
}
// what the values times that power of two are multiplied by
__device__ __forceinline__ float rms_factor(float mean_square, float eps, float scale) { return 1.0f / sqrtf(mean_square + eps * scale * scale); }

// The scale of a row whose largest |y| has the bits `most`, and what y is multiplied by, twice, to become q: one factor would leave float32's
// range for the smallest rows. Bits from those of infinity on: not every value is finite.
struct RowScale { float scale, first, second; };
__device__ __forceinline__ RowScale row_scale(uint32_t most) {
    if (most >= 0x7f800000u) return {__builtin_nanf(""), 0.0f, 0.0f};
    const float m = __builtin_bit_cast(float, most);
    if (m == 0.0f) return {0.0f, 0.0f, 0.0f};
    const float first = m < 0x1p-100f ? 0x1p100f : 1.0f;
    return {m / 127.0f, first, 127.0f / (m * first)};
}
__device__ __forceinline__ int8_t eight_bits(float y, const RowScale& s) {
    const float q = rintf(y * s.first * s.second);
    return s.second == 0.0f ? (int8_t)0 : (int8_t)(int)fminf(fmaxf(q, -127.0f), 127.0f);
}

template <class T, int TH, int NV>
__global__ __launch_bounds__(TH < 256 ? 256 : TH) void rms_norm_rows(RmsArgs p) {
    constexpr int E = 16 / sizeof(T), ROWS = TH < 256 ? 256 / TH : 1;
    __shared__ float part_sum[2][16];
    __shared__ uint32_t part_max[16];
    const int t = threadIdx.x % TH;
    int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TH;
    const bool mine = row < p.rows;
    if (!mine) row = p.rows - 1;   // (barriers below are for every thread)
    const T* x = static_cast<const T*>(p.X) + row * p.cols;
    const T* skip = p.skip ? static_cast<const T*>(p.skip) + row * p.cols : nullptr;
    const int cols = (int)p.cols;

    float v[NV][E];
#pragma unroll
    for (int j = 0; j < NV; ++j) load_values(v[j], x + (t + j * TH) * E, cols - (t + j * TH) * E);
    if (skip) {
        float s[NV][E];
#pragma unroll
        for (int j = 0; j < NV; ++j) load_values(s[j], skip + (t + j * TH) * E, cols - (t + j * TH) * E);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) v[j][e] += s[j][e];
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) sum = fmaf(v[j][e], v[j][e], sum);
    const float n = (float)cols;
    float mean = threads_sum<TH>(sum, part_sum[0]) / n;
    const float scale = rms_rescale(mean, p.eps);
    if (scale != 1.0f) {   // (the same for all threads of a barrier)
        sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) sum = fmaf(v[j][e] * scale, v[j][e] * scale, sum);
        mean = threads_sum<TH>(sum, part_sum[1]) / n;
    }
    const float factor = rms_factor(mean, p.eps, scale);

    if (p.Sum && mine) {
        T* to = static_cast<T*>(p.Sum) + row * p.cols;
#pragma unroll
        for (int j = 0; j < NV; ++j) store_values(to + (t + j * TH) * E, v[j], cols - (t + j * TH) * E);
    }
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float g[E];
        load_values(g, static_cast<const T*>(p.gain) + (t + j * TH) * E, cols - (t + j * TH) * E);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[j][e] = v[j][e] * scale * factor * g[e];
            const bool inside = (t + j * TH) * E + e < cols;   // (0 times an infinite factor outside)
            const uint32_t bits = inside ? __builtin_bit_cast(uint32_t, v[j][e]) & 0x7fffffffu : 0u;
            most = most > bits ? most : bits;
        }
    }
    if (p.Y && mine) {
        T* to = static_cast<T*>(p.Y) + row * p.cols;
#pragma unroll
        for (int j = 0; j < NV; ++j) store_values(to + (t + j * TH) * E, v[j], cols - (t + j * TH) * E);
    }
    if (p.Q) {
        const RowScale s = row_scale(threads_max<TH>(most, part_max));
        if (mine) {
            int8_t* to = p.Q + row * p.cols;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                int8_t q[E];
#pragma unroll
                for (int e = 0; e < E; ++e) q[e] = eight_bits(v[j][e], s);
                store_values(to + (t + j * TH) * E, q, cols - (t + j * TH) * E);
            }
            if (t == 0) p.q_scale[row] = s.scale;
        }
    }
}

template <class T>
__global__ __launch_bounds__(1024) void rms_norm_long(RmsArgs p) {
    constexpr int TH = 1024;
    __shared__ float part_sum[2][16];
    __shared__ uint32_t part_max[16];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.X) + row * p.cols;
    const T* skip = p.skip ? static_cast<const T*>(p.skip) + row * p.cols : nullptr;
    const T* gain = static_cast<const T*>(p.gain);
    auto value = [&](int64_t c) { return skip ? (float)x[c] + (float)skip[c] : (float)x[c]; };

    float sum = 0.0f;
    for (int64_t c = threadIdx.x; c < p.cols; c += TH) sum = fmaf(value(c), value(c), sum);
    float mean = threads_sum<TH>(sum, part_sum[0]) / (float)p.cols;
    const float scale = rms_rescale(mean, p.eps);
    if (scale != 1.0f) {   // (the same for all threads)
        sum = 0.0f;
        for (int64_t c = threadIdx.x; c < p.cols; c += TH) sum = fmaf(value(c) * scale, value(c) * scale, sum);
        mean = threads_sum<TH>(sum, part_sum[1]) / (float)p.cols;
    }
    const float factor = rms_factor(mean, p.eps, scale);
    uint32_t most = 0;
    for (int64_t c = threadIdx.x; c < p.cols; c += TH) {
        const float s = value(c), y = s * scale * factor * (float)gain[c];
        const uint32_t bits = __builtin_bit_cast(uint32_t, y) & 0x7fffffffu;
        most = most > bits ? most : bits;
        if (p.Sum) static_cast<T*>(p.Sum)[row * p.cols + c] = (T)s;
        if (p.Y) static_cast<T*>(p.Y)[row * p.cols + c] = (T)y;
    }
    if (p.Q) {
        const RowScale s = row_scale(threads_max<TH>(most, part_max));
        for (int64_t c = threadIdx.x; c < p.cols; c += TH) p.Q[row * p.cols + c] = eight_bits(value(c) * scale * factor * (float)gain[c], s);
        if (threadIdx.x == 0) p.q_scale[row] = s.scale;
    }
}

// false: more workgroups than a launch has
template <class T>
static bool launch_rms_norm(const RmsArgs& p, hipStream_t st) {
    constexpr int64_t E = 16 / sizeof(T);
    bool fits = true;
    auto rows = [&](auto th, auto nv) {
        constexpr int TH = decltype(th)::value, NV = decltype(nv)::value, ROWS = TH < 256 ? 256 / TH : 1, THREADS = TH < 256 ? 256 : TH;
        const int64_t grid = ceil_div(p.rows, (int64_t)ROWS);
        fits = grid_fits(grid, THREADS);
        if (fits) hipLaunchKernelGGL((rms_norm_rows<T, TH, NV>), dim3((unsigned)grid), dim3(THREADS), 0, st, p);
    };
    const int64_t vectors = ceil_div(p.cols, E);
    if (vectors <= 64) rows(Int<64>{}, Int<1>{});
    else if (vectors <= 128) rows(Int<64>{}, Int<2>{});
    else if (vectors <= 256) rows(Int<256>{}, Int<1>{});
    else if (vectors <= 512) rows(Int<256>{}, Int<2>{});
    else if (vectors <= 1024) rows(Int<256>{}, Int<4>{});
    else if (vectors <= 2048) rows(Int<1024>{}, Int<2>{});
    else if (vectors <= 4096) rows(Int<1024>{}, Int<4>{});
    else {
        fits = grid_fits(p.rows, 1024);
        if (fits) hipLaunchKernelGGL(rms_norm_long<T>, dim3((unsigned)p.rows), dim3(1024), 0, st, p);
    }
    return fits;
}

}  // namespace mi355x

extern "C" int mi355x_skip_rms_norm(const void* X, const void* skip, const void* gain, void* Y, void* Sum, int8_t* Q, float* q_scale,
                                    int64_t rows, int64_t cols, int type, float epsilon, void* stream) {
    using namespace mi355x;
    MI355X_REQUIRE(rows >= 0 && cols >= 0, "skip_rms_norm: negative extent (rows=%lld cols=%lld)", (long long)rows, (long long)cols);
    MI355X_REQUIRE(is_mixed_type(type), "skip_rms_norm: element type %d", type);
    MI355X_REQUIRE(epsilon >= 0.0f && epsilon < __builtin_inff(), "skip_rms_norm: epsilon %g", (double)epsilon);
    MI355X_REQUIRE((Q == nullptr) == (q_scale == nullptr), "skip_rms_norm: Q and q_scale go together");
    MI355X_REQUIRE(Y || Sum || Q, "skip_rms_norm: no output");
    MI355X_REQUIRE(rows == 0 || cols > 0, "skip_rms_norm: rows without columns");
    if (rows == 0) return MI355X_OK;
    MI355X_REQUIRE(X && gain, "skip_rms_norm: null pointer (X and gain are required)");
    MI355X_REQUIRE(cols < ((int64_t)1 << 31) - 65536 && rows < (int64_t)1 << 40, "skip_rms_norm: too many rows or columns");
    const bool over = Sum == X || Y == X || (skip && (Sum == skip || Y == skip));
    const int64_t vectors = ceil_div(cols, (int64_t)(type == MI355X_TYPE_FLOAT ? 4 : 8));
    MI355X_REQUIRE(!over || vectors <= 4096, "skip_rms_norm: rows of %lld columns cannot be written over the input", (long long)cols);
    MI355X_REQUIRE(Sum == nullptr || Sum != Y, "skip_rms_norm: Sum and Y are one array");
    const RmsArgs p = {X, skip, gain, Y, Sum, Q, q_scale, rows, cols, epsilon};
    bool fits = true;
    with_type(type, [&](auto t) { fits = launch_rms_norm<decltype(t)>(p, static_cast<hipStream_t>(stream)); });
    MI355X_REQUIRE(fits, "skip_rms_norm: too many rows");
    return check_launch("rms_norm_rows");
}
