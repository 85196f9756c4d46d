// DraftAcceptance: the largest of every row of logits, and the walk along each entry's tree of drafted tokens that follows them. The reference has no such node.
#include "mixed.h"

namespace mi355x {

constexpr int ACCEPT_MOST = 1024;   // tokens of a tree

struct AcceptArgs {
    const void* logits; const int32_t* tokens; const int32_t* parents;
    int32_t* path; int32_t* count; int32_t* next;
    uint64_t* best;   // [rows][parts]: order of the value, then how far the place is from the end
    int64_t rows, vocabulary, part;
    int batch_tokens, parts;
};

// Larger for larger values, the same for 0 and -0; 0 for a NaN
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v + 0.0f);
    return v != v ? 0u : bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ uint64_t wave_largest(uint64_t v) {
#pragma unroll
    for (int d = 32; d; d /= 2) v = larger(v, __shfl_xor(v, d));
    return v;
}

template <class T>
__global__ __launch_bounds__(256) void accept_rows_kernel(AcceptArgs p) {
    __shared__ uint64_t found[4];
    const int64_t row = blockIdx.x / p.parts, first = blockIdx.x % p.parts * p.part;
    const int64_t last = first + p.part < p.vocabulary ? first + p.part : p.vocabulary;
    const T* x = static_cast<const T*>(p.logits) + row * p.vocabulary;
    uint64_t best = 0;
    for (int64_t i = first + threadIdx.x; i < last; i += 256) best = larger(best, (uint64_t)order_of((float)x[i]) << 32 | (uint32_t)~(uint32_t)i);
    best = wave_largest(best);
    if (threadIdx.x % WAVE == 0) found[threadIdx.x / WAVE] = best;
    __syncthreads();
    if (threadIdx.x == 0) p.best[blockIdx.x] = larger(larger(found[0], found[1]), larger(found[2], found[3]));
}

// A workgroup to an entry. A token's children stand behind it, so one pass over the tokens finds the whole path.
__global__ __launch_bounds__(256) void accept_walk_kernel(AcceptArgs p) {
    __shared__ int32_t said[ACCEPT_MOST], tokens[ACCEPT_MOST], parents[ACCEPT_MOST];
    const int S = p.batch_tokens;
    const int64_t row0 = (int64_t)blockIdx.x * S;
    for (int i = threadIdx.x; i < S; i += 256) {
        uint64_t best = 0;
        for (int c = 0; c < p.parts; ++c) best = larger(best, p.best[(row0 + i) * p.parts + c]);
        said[i] = (int32_t)~(uint32_t)best;
        tokens[i] = p.tokens[row0 + i];
        parents[i] = p.parents ? p.parents[row0 + i] : i - 1;
    }
    __syncthreads();
    if (threadIdx.x) return;
    int node = 0, length = 1;
    p.path[row0] = 0;
    for (int i = 1; i < S; ++i)
        if (parents[i] == node && tokens[i] == said[node]) p.path[row0 + length++] = node = i;
    for (int i = length; i < S; ++i) p.path[row0 + i] = -1;
    p.count[blockIdx.x] = length;
    p.next[blockIdx.x] = said[node];
}

static bool accept_fits(int64_t batch, int64_t tokens, int64_t vocabulary) {
    return batch >= 0 && tokens >= 1 && tokens <= ACCEPT_MOST && vocabulary >= 1 && vocabulary < (int64_t)1 << 31 && batch < (int64_t)1 << 31 && (double)batch * tokens * vocabulary < 0x1p45;
}

static int64_t accept_parts(int64_t rows, int64_t vocabulary) { return rows ? 1 : 1; }

}  // namespace mi355x

extern "C" int64_t mi355x_draft_acceptance_scratch(int64_t batch, int64_t tokens, int64_t vocabulary, int type) {
    using namespace mi355x;
    if (!is_mixed_type(type) || !accept_fits(batch, tokens, vocabulary)) return 0;
    return batch * tokens * accept_parts(batch * tokens, vocabulary);
}

extern "C" int mi355x_draft_acceptance(const void* logits, const int32_t* tokens, const int32_t* parents, int32_t* path, int32_t* count, int32_t* next, void* scratch,
                                       int64_t scratch_words, int64_t batch, int64_t token_count, int64_t vocabulary, int type, void* stream) {
    using namespace mi355x;
    MI355X_REQUIRE(is_mixed_type(type), "draft_acceptance: element type %d", type);
    MI355X_REQUIRE(accept_fits(batch, token_count, vocabulary), "draft_acceptance: %lld trees of %lld tokens, vocabulary of %lld (1 to %d tokens)", (long long)batch,
                   (long long)token_count, (long long)vocabulary, ACCEPT_MOST);
    if (batch == 0) return MI355X_OK;
    MI355X_REQUIRE(logits && tokens && path && count && next, "draft_acceptance: null pointer");
    const int64_t rows = batch * token_count, parts = accept_parts(rows, vocabulary);
    MI355X_REQUIRE(scratch && (reinterpret_cast<uintptr_t>(scratch) & 7) == 0 && scratch_words >= rows * parts, "draft_acceptance: scratch memory for %lld words, 8-byte aligned",
                   (long long)(rows * parts));
    MI355X_REQUIRE(grid_fits(rows * parts, 256), "draft_acceptance: too large");
    AcceptArgs p = {logits, tokens, parents, path, count, next, static_cast<uint64_t*>(scratch), rows, vocabulary, ceil_div(vocabulary, parts), (int)token_count, (int)parts};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    with_type(type, [&](auto t) { hipLaunchKernelGGL((accept_rows_kernel<decltype(t)>), dim3((unsigned)(rows * parts)), dim3(256), 0, st, p); });
    hipLaunchKernelGGL(accept_walk_kernel, dim3((unsigned)batch), dim3(256), 0, st, p);
    return check_launch("draft_acceptance");
}
