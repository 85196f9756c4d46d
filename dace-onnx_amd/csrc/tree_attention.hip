// TreeAttention: O = softmax(c Q K^T) V over a cache in pages, whose last tokens are a chain or a tree. The reference has no such node.
#include "mixed.h"

namespace mi355x {

constexpr int TREE_MOST = 1024;   // tokens of a tree

struct TreeArgs {
    const void* q; const void* k_pages; const void* v_pages; const int32_t* table; const int32_t* lengths; const int32_t* parents; void* o;
    int64_t batch, tokens, pages, page_size, columns;
    int heads, kv_heads, share;
    float scale_log2;
};

// A wave to a row
template <class T, int D>
__global__ __launch_bounds__(64) void tree_attention_kernel(TreeArgs p) {
    constexpr int E = D / WAVE;
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int head = (int)(row % p.heads);
    const int64_t at = row / p.heads, b = at / p.tokens, token = at % p.tokens;
    const int64_t length = p.lengths[b] < 0 ? 0 : p.lengths[b], capacity = p.columns * p.page_size;
    float q[E], o[E] = {}, top = -__builtin_inff(), sum = 0.0f;
    load_values(q, static_cast<const T*>(p.q) + row * D + lane * E, E);
    auto key = [&](int64_t n) {
        if (n >= capacity) return;
        int64_t page = p.table[b * p.columns + n / p.page_size];
        page = page < 0 ? 0 : page >= p.pages ? p.pages - 1 : page;
        const int64_t offset = ((page * p.kv_heads + head / p.share) * p.page_size + n % p.page_size) * D + lane * E;
        float k[E], v[E], s = 0.0f;
        load_values(k, static_cast<const T*>(p.k_pages) + offset, E);
        load_values(v, static_cast<const T*>(p.v_pages) + offset, E);
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(q[e], k[e], s);
        s = wave_sum(s) * p.scale_log2;
        const float now = fmaxf(top, s), factor = top == now ? 1.0f : __builtin_amdgcn_exp2f(top - now), w = __builtin_amdgcn_exp2f(s - (now == -__builtin_inff() ? 0.0f : now));
        sum = fmaf(sum, factor, w);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], factor, w * v[e]);
        top = now;
    };
    for (int64_t n = 0; n < length && n < capacity; ++n) key(n);
    for (int64_t i = token; i >= 0;) {
        key(length + i);
        const int64_t up = p.parents ? p.parents[b * p.tokens + i] : i - 1;
        i = up < i ? up : -1;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = sum == 0.0f ? 0.0f : o[e] / sum;
    store_values(static_cast<T*>(p.o) + row * D + lane * E, o, E);
}

static bool tree_fits(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t size, int64_t page_size, int64_t columns) {
    return batch >= 0 && tokens >= 0 && heads >= 0 && heads < 1 << 20 && kv_heads >= 1 && heads % kv_heads == 0 && (size == 64 || size == 128 || size == 256) && page_size >= 1 &&
           columns >= 0 && batch < (int64_t)1 << 31 && tokens < (int64_t)1 << 31 && (double)page_size * columns < 0x1p31 - 1024 && (double)batch * tokens * heads < 0x1p40;
}

}  // namespace mi355x

extern "C" int64_t mi355x_tree_attention_scratch(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t size, int64_t page_size, int64_t columns, int type) {
    return 0;
}

extern "C" int mi355x_tree_attention(const void* Q, const void* k_pages, const void* v_pages, const int32_t* table, const int32_t* lengths, const int32_t* parents, void* O,
                                     float* scratch, int64_t scratch_floats, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t size, int64_t pages,
                                     int64_t page_size, int64_t columns, float scale, int type, void* stream) {
    using namespace mi355x;
    MI355X_REQUIRE(is_mixed_type(type), "tree_attention: element type %d", type);
    MI355X_REQUIRE(size == 64 || size == 128 || size == 256, "tree_attention: head size %lld (64, 128 and 256 are supported)", (long long)size);
    MI355X_REQUIRE(heads >= 0 && kv_heads >= 1 && heads % kv_heads == 0, "tree_attention: %lld heads share keys and values in %lld groups", (long long)heads, (long long)kv_heads);
    MI355X_REQUIRE(scale > 0.0f && scale < __builtin_inff(), "tree_attention: scale %g (a positive number is needed)", (double)scale);
    MI355X_REQUIRE(!parents || tokens <= TREE_MOST, "tree_attention: a tree of %lld tokens (%d at most)", (long long)tokens, TREE_MOST);
    MI355X_REQUIRE(tree_fits(batch, tokens, heads, kv_heads, size, page_size, columns) && pages >= 1 && pages < (int64_t)1 << 31 &&
                       (double)pages * page_size * kv_heads < 0x1p46, "tree_attention: negative, empty or too large an extent");
    if (batch == 0 || tokens == 0 || heads == 0) return MI355X_OK;
    MI355X_REQUIRE(Q && O && k_pages && v_pages && lengths && (columns == 0 || table), "tree_attention: null pointer");
    MI355X_REQUIRE(((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) == 0, "tree_attention: pages have to stand at 16-byte boundaries");
    TreeArgs p = {Q, k_pages, v_pages, table, lengths, parents, O, batch, tokens, pages, page_size, columns, (int)heads, (int)kv_heads, (int)(heads / kv_heads),
                  scale * 1.44269504088896340736f};
    MI355X_REQUIRE(grid_fits(batch * tokens * heads, 64), "tree_attention: too large");
    with_type(type, [&](auto t) {
        using T = decltype(t);
        const dim3 grid((unsigned)(batch * tokens * heads)), block(64);
        const hipStream_t st = static_cast<hipStream_t>(stream);
        if (size == 64) hipLaunchKernelGGL((tree_attention_kernel<T, 64>), grid, block, 0, st, p);
        else if (size == 128) hipLaunchKernelGGL((tree_attention_kernel<T, 128>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((tree_attention_kernel<T, 256>), grid, block, 0, st, p);
    });
    return check_launch("tree_attention_kernel");
}
