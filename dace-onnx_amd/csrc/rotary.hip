// RotaryPositions: pair i of every head of a token is turned by positions[axis(i)][token] * frequencies[i]; `sections` gives each axis (time,
// height, width) a run of the pairs. Queries and keys in one launch, arrays in float32, float16 or bfloat16, computed in float32. The reference has
// no such node.
//
// An angle is an integer position times a float32 frequency, in float64: exact for positions below 2^29, rounded from there on. It is counted in turns, by a rounded
// factor, and brought into one turn there: off by less than 2^-51 of the turns in all (position 2^40 at frequency 1: 5e-4 radians). Positions far into a context
// are thousands of turns, of which float32 would leave few right digits (position 100000: 0.004 radians). What is left is rounded to float32, pi 2^-24 of an angle at most, and its
// cosine and sine are float32: float32 results are off by 4.9e-8 in the 2-norm, where cosine and sine taken in float64 give 3.6e-8.
// A workgroup has a few tokens: their angles are computed once, into LDS, and then serve all heads. Four tokens keep enough loads of a thread in flight and leave the
// angles' float64 hidden behind other workgroups' bytes. Bound by the bytes of the heads: 32768 tokens of 16 + 4 heads of 128 in bfloat16 61 us, 5.5 TB/s (a copy of 1
// GiB 5.1); 4616 tokens of 12 heads of 64, 48 of them turned, in float32 7.6 us. One token to a request, 8 x 40 heads: 4.4 us by two workgroups of four
// tokens, whose threads go through the heads in five rounds; few tokens are not dealt to more workgroups.
#include "mixed.h"

#include <algorithm>

namespace mi355x {

constexpr int ROTARY_MAX_AXES = 8, ROTARY_THREADS = 256, ROTARY_LDS_ANGLES = 2048;

struct RotaryArgs {
    const void* q; const void* k; const void* positions; const float* frequencies;
    void* q_out; void* k_out;
    int64_t tokens;
    int heads, kv_heads, size, rotated, axes, tokens_per_wg;
    int end[ROTARY_MAX_AXES];   // one past the last pair of each axis
    int wide_positions;         // 64 bits, not 32
};

// VEC pairs to a thread and step. Each step reads what it writes before it writes it: the outputs may be the inputs.
template <class T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(ROTARY_THREADS) void rotary_positions_kernel(RotaryArgs p) {
    __shared__ float2 turn[ROTARY_LDS_ANGLES];
    const int64_t token0 = (int64_t)blockIdx.x * p.tokens_per_wg;
    const int tokens = (int)(p.tokens - token0 < p.tokens_per_wg ? p.tokens - token0 : p.tokens_per_wg);
    const int pairs = p.rotated / 2;

    for (int i = threadIdx.x; i < tokens * pairs; i += ROTARY_THREADS) {
        const int token = i / pairs, pair = i % pairs;
        int axis = 0;
        while (axis + 1 < p.axes && pair >= p.end[axis]) ++axis;
        const int64_t at = axis * p.tokens + token0 + token;
        const int64_t position = p.wide_positions ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
        const double turns = (double)position * (double)p.frequencies[pair] * 0.15915494309189533577;
        float sine, cosine;
        sincospif((float)(2.0 * (turns - rint(turns))), &sine, &cosine);
        turn[i] = make_float2(cosine, sine);
    }
    __syncthreads();

    const int copied = p.size - p.rotated;
    const int turning = pairs / VEC, steps = turning + (copied + 2 * VEC - 1) / (2 * VEC);   // of a head
    const int all_heads = p.heads + p.kv_heads;
    for (int i = threadIdx.x; i < tokens * all_heads * steps; i += ROTARY_THREADS) {
        const int step = i % steps, head = i / steps % all_heads, token = i / steps / all_heads;
        const bool key = head >= p.heads;
        const int64_t offset = (key ? (token0 + token) * p.kv_heads + head - p.heads : (token0 + token) * p.heads + head) * p.size;
        const T* x = static_cast<const T*>(key ? p.k : p.q) + offset;
        T* y = static_cast<T*>(key ? p.k_out : p.q_out) + offset;
        if (step >= turning) {   // values that are not turned, bit by bit
            typedef typename Values<T, 2 * VEC>::unaligned Vector;
            const int c0 = p.rotated + (step - turning) * 2 * VEC;
            if (c0 + 2 * VEC <= p.size) {
                *reinterpret_cast<Vector*>(y + c0) = *reinterpret_cast<const Vector*>(x + c0);
            } else {
                T v[2 * VEC];
#pragma unroll
                for (int e = 0; e < 2 * VEC; ++e)
                    if (c0 + e < p.size) v[e] = x[c0 + e];
#pragma unroll
                for (int e = 0; e < 2 * VEC; ++e)
                    if (c0 + e < p.size) y[c0 + e] = v[e];
            }
            continue;
        }
        const int pair = step * VEC;
        const float2* at = turn + token * pairs + pair;
        float a[VEC], b[VEC];
        if constexpr (INTERLEAVED) {
            float both[2 * VEC];
            load_values(both, x + 2 * pair, 2 * VEC);
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] = both[2 * e], b[e] = both[2 * e + 1];
        } else {
            load_values(a, x + pair, VEC);
            load_values(b, x + pairs + pair, VEC);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float cosine = at[e].x, sine = at[e].y, first = a[e];
            a[e] = first * cosine - b[e] * sine;
            b[e] = b[e] * cosine + first * sine;
        }
        if constexpr (INTERLEAVED) {
            float both[2 * VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) both[2 * e] = a[e], both[2 * e + 1] = b[e];
            store_values(y + 2 * pair, both, 2 * VEC);
        } else {
            store_values(y + pair, a, VEC);
            store_values(y + pairs + pair, b, VEC);
        }
    }
}

template <class T>
static void launch_rotary(const RotaryArgs& p, bool interleaved, hipStream_t st) {
    const int pairs = p.rotated / 2;
    const dim3 grid((unsigned)ceil_div(p.tokens, (int64_t)p.tokens_per_wg)), block(ROTARY_THREADS);
    auto launch = [&](auto vec) {
        constexpr int VEC = decltype(vec)::value;
        if (interleaved) hipLaunchKernelGGL((rotary_positions_kernel<T, VEC, true>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((rotary_positions_kernel<T, VEC, false>), grid, block, 0, st, p);
    };
    if (sizeof(T) == 2 && pairs % 8 == 0) launch(Int<8>{});
    else if (pairs % 4 == 0) launch(Int<4>{});
    else if (pairs % 2 == 0) launch(Int<2>{});
    else launch(Int<1>{});
}

}  // namespace mi355x

extern "C" int mi355x_rotary_positions(const void* Q, const void* K, const void* positions, const float* frequencies, void* Q_out, void* K_out,
                                       int64_t tokens, int64_t heads, int64_t kv_heads, int64_t size, int64_t rotated, int64_t axes,
                                       const int64_t* sections, int interleaved, int position_bytes, int type, void* stream) {
    using namespace mi355x;
    MI355X_REQUIRE(tokens >= 0 && heads >= 0 && kv_heads >= 0 && size >= 0, "rotary_positions: negative extent");
    MI355X_REQUIRE(is_mixed_type(type), "rotary_positions: element type %d", type);
    MI355X_REQUIRE(position_bytes == 4 || position_bytes == 8, "rotary_positions: positions of %d bytes", position_bytes);
    MI355X_REQUIRE(rotated >= 0 && rotated % 2 == 0 && rotated <= size, "rotary_positions: %lld of %lld values", (long long)rotated, (long long)size);
    MI355X_REQUIRE(axes >= 1 && axes <= ROTARY_MAX_AXES && sections, "rotary_positions: %lld axes (1 to %d)", (long long)axes, ROTARY_MAX_AXES);
    MI355X_REQUIRE(rotated / 2 <= ROTARY_LDS_ANGLES && size <= 1 << 16 && heads <= 1 << 12 && kv_heads <= 1 << 12, "rotary_positions: head too large, or too many");
    RotaryArgs p = {Q, K, positions, frequencies, Q_out, K_out, tokens, (int)heads, (int)kv_heads, (int)size, (int)rotated, (int)axes, 1, {}, position_bytes == 8};
    int64_t pairs = 0;
    for (int64_t a = 0; a < axes; ++a) {
        MI355X_REQUIRE(sections[a] >= 0 && sections[a] <= rotated / 2, "rotary_positions: section of %lld pairs", (long long)sections[a]);
        p.end[a] = (int)(pairs += sections[a]);
    }
    MI355X_REQUIRE(pairs == rotated / 2, "rotary_positions: sections of %lld pairs, %lld are turned", (long long)pairs, (long long)(rotated / 2));
    if (tokens == 0 || heads + kv_heads == 0 || size == 0) return MI355X_OK;
    MI355X_REQUIRE((heads == 0 || (Q && Q_out)) && (kv_heads == 0 || (K && K_out)) && (rotated == 0 || (positions && frequencies)), "rotary_positions: null pointer");
    p.tokens_per_wg = std::max(1, std::min(4, ROTARY_LDS_ANGLES / std::max(p.rotated / 2, 1)));
    MI355X_REQUIRE(tokens < (int64_t)1 << 40 && grid_fits(ceil_div(tokens, (int64_t)p.tokens_per_wg), ROTARY_THREADS), "rotary_positions: too many tokens");
    with_type(type, [&](auto t) { launch_rotary<decltype(t)>(p, interleaved != 0, static_cast<hipStream_t>(stream)); });
    return check_launch("rotary_positions_kernel");
}
