// PagedCacheAppend: the keys and values of a call's tokens to their rows of a cache in pages; keys, and the call's queries, turned by the tokens' positions on the way.
// Arrays in float32, float16 or bfloat16, turned in float32. The reference has no such node.
//
// Token j of entry b becomes number n = lengths[b] + j of the entry: row n % page of page table[b, n / page], whatever order the pages were handed out in. Pair i of a head is turned
// by position * frequencies[i] (rotary.h). A workgroup has a few tokens, whose places and angles are found once, into LDS, and then serve their heads.
// Bound by the bytes of the heads: 16384 tokens of 32 + 2 x 8 heads of 128 in bfloat16 79 us, 5.1 TB/s (a copy of 1 GiB 5.1); with few tokens by three reads that need each other (a
// length, the page, the values) and the launch: 16 tokens 4.2 us, 225 tokens of 2 x 6 heads of 64 in float32 4.4.
#include "mixed.h"
#include "rotary.h"

#include <algorithm>

namespace mi355x {

constexpr int APPEND_THREADS = 256, APPEND_TOKENS = 4;

struct AppendArgs {
    const void* k; const void* v; const void* q; void* k_pages; void* v_pages; void* q_out;
    const int32_t* table; const int32_t* lengths; const float* frequencies; const void* positions; const int32_t* order;
    int64_t all, tokens, taken, pages, page_size, columns;   // all = batch * taken
    int64_t per_axis;                                        // batch * tokens
    int heads, kv_heads, size, rotated, axes, tokens_per_wg, heads_per_wg;
    int end[ROTARY_MAX_AXES];   // one past the last pair of each axis
    int wide_positions;         // 64 bits, not 32
};

// Where a token comes from and goes to: source < 0 or page < 0: nowhere
struct AppendPlace {
    int64_t source, number;
    int32_t page, row;
};

__device__ __forceinline__ AppendPlace append_source(const AppendArgs& p, int64_t at) {
    const int64_t b = at / p.taken, j = at % p.taken, length = p.lengths[b], i = p.order ? p.order[at] : j;
    return {i >= 0 && i < p.tokens ? b * p.tokens + i : -1, (length < 0 ? 0 : length) + j, -1, 0};
}

__device__ __forceinline__ AppendPlace append_place(const AppendArgs& p, int64_t at) {
    AppendPlace place = append_source(p, at);
    const int64_t column = place.number / p.page_size;
    if (column < p.columns) {
        const int32_t page = p.table[at / p.taken * p.columns + column];
        if (page >= 0 && page < p.pages) place.page = page;
        place.row = (int32_t)(place.number - column * p.page_size);
    }
    return place;
}

// n values of x to y, bit by bit
template <class T, int N>
__device__ __forceinline__ void copy_values(T* y, const T* x, int n) {
    typedef typename Values<T, N>::unaligned Vector;
    if (n >= N) {
        *reinterpret_cast<Vector*>(y) = *reinterpret_cast<const Vector*>(x);
        return;
    }
    T v[N];
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e < n) v[e] = x[e];
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e < n) y[e] = v[e];
}

// VEC pairs, or 2 VEC values that are copied, to a thread and step. Each step reads what it writes before it writes it: Q_out may be Q.
template <class T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(APPEND_THREADS) void paged_append_kernel(AppendArgs p) {
    __shared__ float2 turn[ROTARY_LDS_ANGLES];
    __shared__ AppendPlace places[APPEND_TOKENS];
    const int64_t token0 = (int64_t)blockIdx.x * p.tokens_per_wg;
    const int tokens = (int)(p.all - token0 < p.tokens_per_wg ? p.all - token0 : p.tokens_per_wg);
    const int pairs = p.rotated / 2;
    // Places and angles at once: a thread that takes an angle looks for the token's number itself rather than wait for the one that looks into the table.
    if ((int)threadIdx.x < tokens) places[threadIdx.x] = append_place(p, token0 + threadIdx.x);
    for (int i = threadIdx.x; i < tokens * pairs; i += APPEND_THREADS) {
        const int token = i / pairs, pair = i % pairs;
        const float frequency = p.frequencies[pair];
        const AppendPlace place = append_source(p, token0 + token);
        if (place.source < 0) continue;
        int64_t position = place.number;
        if (p.positions) {
            int axis = 0;
            while (axis + 1 < p.axes && pair >= p.end[axis]) ++axis;
            const int64_t at = axis * p.per_axis + place.source;
            position = p.wide_positions ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
        }
        turn[i] = rotary_turn(position, frequency);
    }
    __syncthreads();

    const int copied = p.size - p.rotated;
    const int turning = pairs / VEC, steps = turning + (copied + 2 * VEC - 1) / (2 * VEC);   // of a head; of one that is copied whole no more
    const int all_heads = p.heads + 2 * p.kv_heads, head0 = blockIdx.y * p.heads_per_wg, my_heads = min(p.heads_per_wg, all_heads - head0);
    for (int i = threadIdx.x; i < tokens * my_heads * steps; i += APPEND_THREADS) {
        const int step = i % steps, head = head0 + i / steps % my_heads, token = i / steps / my_heads;
        const AppendPlace& place = places[token];
        if (place.source < 0 || (head >= p.heads && place.page < 0)) continue;
        const T* x;
        T* y;
        const bool value = head >= p.heads + p.kv_heads;
        if (head < p.heads) {
            const int64_t offset = (place.source * p.heads + head) * p.size;
            x = static_cast<const T*>(p.q) + offset;
            y = static_cast<T*>(p.q_out) + offset;
        } else {
            const int g = head - p.heads - (value ? p.kv_heads : 0);
            x = static_cast<const T*>(value ? p.v : p.k) + (place.source * p.kv_heads + g) * p.size;
            y = static_cast<T*>(value ? p.v_pages : p.k_pages) + (((int64_t)place.page * p.kv_heads + g) * p.page_size + place.row) * p.size;
        }
        if (value || step >= turning) {
            const int c0 = value ? step * 2 * VEC : p.rotated + (step - turning) * 2 * VEC;
            copy_values<T, 2 * VEC>(y + c0, x + c0, p.size - c0);
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
static void launch_append(AppendArgs p, bool interleaved, hipStream_t st) {
    const int pairs = p.rotated / 2;
    const dim3 block(APPEND_THREADS);
    auto launch = [&](auto vec) {
        constexpr int VEC = decltype(vec)::value;
        // Few tokens: one to a workgroup, and no more of its heads than its threads have a step of. Otherwise four tokens share what is found out about pages and angles. us, tokens of
        // 32 + 2 x 8 heads of 128, four whole ones / shares of one: 16 in bfloat16 6.4 / 4.2 (the kernel alone); with the call around it: 512 in float32 12.2 / 7.8, 1024 in bfloat16 9.6 / 8.4,
        // 2048 11.4 / 13.0, 4096 17.9 / 21.2.
        const int all_heads = p.heads + 2 * p.kv_heads, steps = (p.size + 2 * VEC - 1) / (2 * VEC);
        p.heads_per_wg = all_heads;
        if (p.all <= 1024) {
            p.tokens_per_wg = 1;
            p.heads_per_wg = std::min(all_heads, std::max(1, APPEND_THREADS / std::max(steps, 1)));
        }
        const dim3 grid((unsigned)ceil_div(p.all, (int64_t)p.tokens_per_wg), (unsigned)ceil_div((int64_t)all_heads, (int64_t)p.heads_per_wg));
        if (interleaved) hipLaunchKernelGGL((paged_append_kernel<T, VEC, true>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((paged_append_kernel<T, VEC, false>), grid, block, 0, st, p);
    };
    if (sizeof(T) == 2 && pairs % 8 == 0) launch(Int<8>{});
    else if (pairs % 4 == 0) launch(Int<4>{});
    else if (pairs % 2 == 0) launch(Int<2>{});
    else launch(Int<1>{});
}

}  // namespace mi355x

extern "C" int mi355x_paged_cache_append(const void* K, const void* V, const void* Q, void* k_pages, void* v_pages, void* Q_out, const int32_t* table,
                                         const int32_t* lengths, const float* frequencies, const void* positions, const int32_t* order, int64_t batch,
                                         int64_t tokens, int64_t heads, int64_t kv_heads, int64_t size, int64_t pages, int64_t page_size, int64_t columns,
                                         int64_t taken, int64_t rotated, int64_t axes, const int64_t* sections, int interleaved, int position_bytes, int type,
                                         void* stream) {
    using namespace mi355x;
    MI355X_REQUIRE(batch >= 0 && tokens >= 0 && heads >= 0 && kv_heads >= 0 && size >= 0 && pages >= 0 && columns >= 0 && taken >= 0, "paged_cache_append: negative extent");
    MI355X_REQUIRE(is_mixed_type(type), "paged_cache_append: element type %d", type);
    MI355X_REQUIRE(page_size >= 1, "paged_cache_append: pages of %lld", (long long)page_size);
    MI355X_REQUIRE(position_bytes == 4 || position_bytes == 8, "paged_cache_append: positions of %d bytes", position_bytes);
    MI355X_REQUIRE(rotated >= 0 && rotated % 2 == 0 && rotated <= size, "paged_cache_append: %lld of %lld values", (long long)rotated, (long long)size);
    MI355X_REQUIRE(axes >= 1 && axes <= ROTARY_MAX_AXES && sections, "paged_cache_append: %lld axes (1 to %d)", (long long)axes, ROTARY_MAX_AXES);
    MI355X_REQUIRE(axes == 1 || positions, "paged_cache_append: a token's own number is one axis, not %lld", (long long)axes);
    MI355X_REQUIRE(heads == 0 || !order, "paged_cache_append: queries are turned in their own order");
    MI355X_REQUIRE(order || taken == tokens || taken == 0, "paged_cache_append: %lld of %lld tokens without an order", (long long)taken, (long long)tokens);
    MI355X_REQUIRE(rotated / 2 <= ROTARY_LDS_ANGLES && size <= 1 << 16 && heads <= 1 << 12 && kv_heads <= 1 << 12, "paged_cache_append: head too large, or too many");
    MI355X_REQUIRE(batch < (int64_t)1 << 31 && tokens < (int64_t)1 << 31 && taken < (int64_t)1 << 31 && pages < (int64_t)1 << 31 && page_size < (int64_t)1 << 31 &&
                       columns < (int64_t)1 << 31, "paged_cache_append: too large");
    AppendArgs p = {K, V, Q, k_pages, v_pages, Q_out, table, lengths, frequencies, positions, order, batch * taken, tokens, taken, pages, page_size, columns, batch * tokens,
                    (int)heads, (int)kv_heads, (int)size, (int)rotated, (int)axes, 1, 1, {}, position_bytes == 8};
    int64_t pairs = 0;
    for (int64_t a = 0; a < axes; ++a) {
        MI355X_REQUIRE(sections[a] >= 0 && sections[a] <= rotated / 2, "paged_cache_append: section of %lld pairs", (long long)sections[a]);
        p.end[a] = (int)(pairs += sections[a]);
    }
    MI355X_REQUIRE(pairs == rotated / 2, "paged_cache_append: sections of %lld pairs, %lld are turned", (long long)pairs, (long long)(rotated / 2));
    if (p.all == 0 || heads + kv_heads == 0 || size == 0) return MI355X_OK;
    MI355X_REQUIRE(lengths && (columns == 0 || table) && (heads == 0 || (Q && Q_out)) && (rotated == 0 || frequencies), "paged_cache_append: null pointer");
    MI355X_REQUIRE(kv_heads == 0 || ((tokens == 0 || (K && V)) && (pages == 0 || (k_pages && v_pages))), "paged_cache_append: null pointer");
    p.tokens_per_wg = std::max(1, std::min(APPEND_TOKENS, ROTARY_LDS_ANGLES / std::max(p.rotated / 2, 1)));
    MI355X_REQUIRE(p.all < (int64_t)1 << 40 && p.per_axis < (int64_t)1 << 40 && (double)pages * page_size * kv_heads < 0x1p46 &&
                       grid_fits(ceil_div(p.all, (int64_t)p.tokens_per_wg), APPEND_THREADS), "paged_cache_append: too many tokens");
    const uint64_t at_k = reinterpret_cast<uint64_t>(k_pages), at_v = reinterpret_cast<uint64_t>(v_pages), apart = (at_k < at_v ? at_v - at_k : at_k - at_v) / (type == MI355X_TYPE_FLOAT ? 4 : 2);
    MI355X_REQUIRE(apart >= (uint64_t)(pages * kv_heads * page_size * size), "paged_cache_append: keys and values share pages");
    with_type(type, [&](auto t) { launch_append<decltype(t)>(p, interleaved != 0, static_cast<hipStream_t>(stream)); });
    return check_launch("paged_append_kernel");
}
