// DraftAcceptance: the largest of every row of logits, and the walk along each entry's tree of drafted tokens that follows them. The reference has no such node.
//
// Every row is looked at, also those that the walk does not come to: which they are is known only once the largest of the rows before are, and reading all at once is one pass over memory. A
// row's largest is that of its parts' keys, in 64 bits: the value's order, then how far its place is from the row's end, so the first of equal ones wins in any order of the parts, and nothing
// has to be cleared or added to by atomics. Values are compared as they are; nothing is rounded.
// Bound by the bytes of the logits: 16 trees of 32 over 131072 in bfloat16 25 to 26 us, 5.3 TB/s, and 3.9 for the walk. 8 rows of 32000: 3.4 and 2.2 us, less than the host
// takes for the call (10.3).
#include "mixed.h"

#include <algorithm>

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

// A part of a row to a workgroup. A thread keeps the vector that has the largest of its values, the first of equal ones, and looks for the place in it at the end.
template <class T>
__global__ __launch_bounds__(256) void accept_rows_kernel(AcceptArgs p) {
    constexpr int E = 16 / sizeof(T), AHEAD = 4;
    typedef typename Values<T, E>::vec Vector;
    __shared__ uint64_t found[4];
    const int64_t row = blockIdx.x / p.parts, first = blockIdx.x % p.parts * p.part;
    const int64_t last = first + p.part < p.vocabulary ? first + p.part : p.vocabulary;
    const T* x = static_cast<const T*>(p.logits) + row * p.vocabulary;
    auto key = [](uint32_t order, int64_t place) { return (uint64_t)order << 32 | (uint32_t)~(uint32_t)place; };
    // vectors begin at 16-byte boundaries; what stands before and behind them goes by single values
    const int64_t gap = (int64_t)((16 - (reinterpret_cast<uintptr_t>(x + first) & 15)) & 15) / (int64_t)sizeof(T);
    const int64_t begin = first + gap < last ? first + gap : last, vectors = (last - begin) / E, end = begin + vectors * E;
    uint64_t best = 0;
    const int64_t single = (int64_t)threadIdx.x < begin - first ? first + threadIdx.x : (int64_t)threadIdx.x - E < last - end && threadIdx.x >= E ? end + threadIdx.x - E : -1;
    if (single >= 0) best = key(order_of((float)x[single]), single);
    const Vector* v = reinterpret_cast<const Vector*>(x + begin);
    uint32_t largest = 0;
    int64_t which = threadIdx.x;
    Vector kept = {};
    for (int64_t i0 = threadIdx.x; i0 < vectors; i0 += 256 * AHEAD) {
        Vector held[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) held[u] = v[i0 + 256 * u < vectors ? i0 + 256 * u : i0];   // (again the first, where there is none: not larger than itself)
        if (i0 == threadIdx.x) kept = held[0];   // (of NaN only: the first of them)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            float m = (float)held[u][0];
#pragma unroll
            for (int e = 1; e < E; ++e) m = fmaxf(m, (float)held[u][e]);
            const uint32_t order = order_of(m);
            if (order > largest) largest = order, which = i0 + 256 * u, kept = held[u];
        }
    }
    if ((int64_t)threadIdx.x < vectors) {
        int place = 0;
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
            if (order_of((float)kept[e]) == largest) place = e;
        best = larger(best, key(largest, begin + which * E + place));
    }
    best = wave_largest(best);
    if (threadIdx.x % WAVE == 0) found[threadIdx.x / WAVE] = best;
    __syncthreads();
    if (threadIdx.x == 0) p.best[blockIdx.x] = larger(larger(found[0], found[1]), larger(found[2], found[3]));
}

// What the logits of a row say
__device__ __forceinline__ int32_t accept_said(const AcceptArgs& p, int64_t row) {
    uint64_t best = 0;
#pragma unroll 8
    for (int c = 0; c < p.parts; ++c) best = larger(best, p.best[row * p.parts + c]);
    return (int32_t)~(uint32_t)best;
}

// Trees of up to 64 tokens, a wave to an entry: a lane has a token, and a step looks at all of them without LDS: 2.2 us for one of 8 where the
// kernel below takes 2.8; a call with 16 of 32 28.7 for 30.0 (the kept vectors of the first kernel included).
__global__ __launch_bounds__(WAVE) void accept_walk_wave_kernel(AcceptArgs p) {
    const int S = p.batch_tokens, i = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * S;
    int32_t token = 0, parent = -1, said = 0, place = -1;
    if (i < S) {
        token = p.tokens[row0 + i];
        parent = p.parents ? p.parents[row0 + i] : i - 1;
        said = accept_said(p, row0 + i);
    }
    int node = 0, length = 0;
    int32_t wanted;
    while (true) {
        place = i == length ? node : place;
        ++length;
        wanted = __builtin_amdgcn_readlane(said, node);
        const uint64_t fits = __ballot(i < S && i > node && parent == node && token == wanted);
        if (!fits) break;
        node = __builtin_ctzll(fits);
    }
    if (i < S) p.path[row0 + i] = place;
    if (i == 0) p.count[blockIdx.x] = length, p.next[blockIdx.x] = wanted;
}

// Larger ones, a workgroup to an entry. A token's children stand behind it: each step looks at the tokens from its own 64 on.
__global__ __launch_bounds__(256) void accept_walk_kernel(AcceptArgs p) {
    __shared__ int32_t said[ACCEPT_MOST], tokens[ACCEPT_MOST], parents[ACCEPT_MOST];
    const int S = p.batch_tokens;
    const int64_t row0 = (int64_t)blockIdx.x * S;
    for (int i = threadIdx.x; i < S; i += 256) {
        const int32_t token = p.tokens[row0 + i], parent = p.parents ? p.parents[row0 + i] : i - 1;
        said[i] = accept_said(p, row0 + i);
        tokens[i] = token;
        parents[i] = parent;
    }
    __syncthreads();
    if (threadIdx.x >= WAVE) return;
    int node = 0, length = 0;
    while (true) {
        if (threadIdx.x == 0) p.path[row0 + length] = node;
        ++length;
        const int32_t wanted = said[node];
        int child = S;
        for (int i0 = node / WAVE * WAVE; i0 < S && child == S; i0 += WAVE) {
            const int i = i0 + threadIdx.x;
            const uint64_t fits = __ballot(i < S && i > node && parents[i] == node && tokens[i] == wanted);
            if (fits) child = i0 + __builtin_ctzll(fits);
        }
        if (child == S) break;
        node = child;
    }
    for (int i = length + threadIdx.x; i < S; i += WAVE) p.path[row0 + i] = -1;
    if (threadIdx.x == 0) p.count[blockIdx.x] = length, p.next[blockIdx.x] = said[node];
}

static bool accept_fits(int64_t batch, int64_t tokens, int64_t vocabulary) {
    return batch >= 0 && tokens >= 1 && tokens <= ACCEPT_MOST && vocabulary >= 1 && vocabulary < (int64_t)1 << 31 && batch < (int64_t)1 << 31 && (double)batch * tokens * vocabulary < 0x1p45;
}

// Workgroups to a row: enough for all CUs several times, none with less than two vectors to a thread (16 bits).
static int64_t accept_parts(int64_t rows, int64_t vocabulary) {
    const int forced = tuning().accept_parts;
    if (forced > 0) return std::min<int64_t>(forced, vocabulary);
    return std::max<int64_t>(1, std::min({ceil_div((int64_t)2048, std::max<int64_t>(rows, 1)), vocabulary / 4096, (int64_t)64}));
}

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
    if (token_count <= WAVE) hipLaunchKernelGGL(accept_walk_wave_kernel, dim3((unsigned)batch), dim3(WAVE), 0, st, p);
    else hipLaunchKernelGGL(accept_walk_kernel, dim3((unsigned)batch), dim3(256), 0, st, p);
    return check_launch("draft_acceptance");
}
