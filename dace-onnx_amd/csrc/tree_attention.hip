// TreeAttention: O = softmax(c Q K^T) V over a cache in pages, whose last tokens are a chain or a tree. The reference has no such node.
#include "attention_tile.h"

#include <algorithm>

namespace mi355x {

constexpr int TREE_MOST = 1024;   // tokens of a tree

struct TreeArgs {
    const void* q; const void* k_pages; const void* v_pages; const int32_t* table; const int32_t* lengths; const int32_t* parents; void* o;
    float* partial_o; float* partial_ml;   // of splits; [split][slice][row][D], [split][slice][row][2]
    int64_t batch, tokens, columns, row_blocks;
    int pages, page_size, capacity;        // capacity = page_size * columns
    int heads, kv_heads, share, splits;    // share = heads / kv_heads
    uint32_t page_magic; int page_shift;   // n / page_size for n below 2^31
    float scale_log2;
};

__device__ __forceinline__ int tree_column(const TreeArgs& p, int n) { return (int)(__umulhi(2u * (uint32_t)n, p.page_magic) >> p.page_shift); }

// the lowest n of 32 bits
__device__ __forceinline__ uint32_t lowest_bits(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }

// Waves: RW blocks of 32 RB rows, KW shares of a stage's keys, 32 SUB each; NS stages.
template <class T, int D, int RB, int RW, int KW, int SUB, int NS, int PER_SIMD>
__global__ __launch_bounds__(64 * RW * KW, PER_SIMD) void tree_attention_kernel(TreeArgs p) {
    using Tile = AttentionTile<T, D>;
    using Wave = AttentionWave<T, D, D>;
    using Piece = typename Wave::Piece;
    using UnalignedPiece = typename Wave::UnalignedPiece;
    constexpr int KT = 32 * KW * SUB, E = Tile::E, NT = 64 * RW * KW, VT = Wave::VT, ROWS = 32 * RB * RW;
    constexpr int HALF = KT * Tile::ROW, STAGE = 2 * HALF;            // keys, then values
    constexpr int PER_T = KT * Tile::PIECES / NT, KPT = WAVE / Tile::PIECES;   // transfers of a wave's keys in a stage, keys to a transfer
    static_assert(KT * Tile::PIECES % NT == 0 && Tile::PIECES <= WAVE && NS >= 2 && (NS - 2) * 2 * PER_T < 64, "whole pieces to a thread, whole keys to a transfer");
    constexpr int EXCHANGE = 32 * D;   // floats of a row block's output
    __shared__ __attribute__((aligned(1024))) unsigned char lds[std::max(NS * STAGE, KW == 1 ? 0 : 4 * EXCHANGE * (KW / 2) * RW * RB)];
    __shared__ int16_t parents[TREE_MOST];
    __shared__ uint32_t odd_keys[2][KT / 32];   // of the stage and the one before

    const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int n = lane % 32, h = lane / 32, row_wave = wave % RW, key_wave = wave / RW;
    const int64_t logical = xcd_remap(blockIdx.x, (int64_t)gridDim.x);
    const int64_t turn = logical % p.row_blocks, rest = logical / p.row_blocks, slice = rest / p.splits;
    const int split = (int)(rest % p.splits);
    const int64_t b = slice / p.kv_heads;
    const int group = (int)(slice % p.kv_heads);
    const int64_t rows = p.tokens * p.share, block = p.row_blocks - 1 - turn;   // long ones first
    const int given = p.lengths[b];
    const int length = given < 0 ? 0 : given > p.capacity ? p.capacity : given;
    const int total = (int)std::min<int64_t>(length + p.tokens, p.capacity);
    // keys up to and with token `row / share`
    auto up_to = [&](int64_t row) { return (int)std::min<int64_t>(total, length + row / p.share + 1); };

    if (tid < KT / 32) odd_keys[0][tid] = odd_keys[1][tid] = 0;
    if (p.parents) {
        for (int i = tid; i < (int)p.tokens; i += NT) {
            const int parent = p.parents[b * p.tokens + i];
            parents[i] = (int16_t)(parent >= 0 && parent < i ? parent : -1);
        }
    }

    // ---- queries: row r of a slice is head r % share of token r / share ------------------------------------
    const int64_t row0 = block * ROWS + row_wave * RB * 32;   // of the wave
    int token[RB], ancestor[RB];
    Operand<T> q[RB][Wave::QP];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        const int64_t row = row0 + 32 * i + n, r = row < rows ? row : rows - 1;
        token[i] = ancestor[i] = (int)(r / p.share);
        const int head = group * p.share + (int)(r % p.share);
        const T* from = static_cast<const T*>(p.q) + ((b * p.tokens + token[i]) * p.heads + head) * D + 8 * h;
#pragma unroll
        for (int s = 0; s < Wave::QP; ++s) {
            T v[8];
#pragma unroll
            for (int j = 0; j < 8 / E; ++j) {
                const Piece piece = *reinterpret_cast<const UnalignedPiece*>(from + 16 * s + j * E);
#pragma unroll
                for (int e = 0; e < E; ++e) v[j * E + e] = piece[e];
            }
            q[i][s].set(v);
        }
    }
    // keys that any row of the workgroup sees, and that all of them see; the same of the wave
    const int end = up_to(std::min(rows, (block + 1) * ROWS) - 1), all = p.parents ? length : up_to(block * ROWS);
    const int wave_end = row0 < rows ? __builtin_amdgcn_readfirstlane(up_to(std::min(rows, row0 + 32 * RB) - 1)) : 0;
    const int wave_all = p.parents ? length : __builtin_amdgcn_readfirstlane(up_to(std::min(rows - 1, row0)));
    const int stages = (end + KT - 1) / KT, per_split = (stages + p.splits - 1) / p.splits;
    const int first = split * per_split, count = std::max(0, std::min(stages, first + per_split) - first), last = first + count;

    // ---- keys and values -----------------------------------------------------------------------------------
    const T* K = static_cast<const T*>(p.k_pages);
    const T* V = static_cast<const T*>(p.v_pages);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds;
    typedef const __attribute__((address_space(4))) int32_t Uniform;   // (read by scalar loads, which the transfers' counter does not count)
    Uniform* const table = (Uniform*)(uintptr_t)(p.table + b * p.columns);
    auto page_at = [&](int column) { return std::min(std::max((int)table[column], 0), p.pages - 1); };
    auto row_at = [&](int page, int row) { return (((int64_t)page * p.kv_heads + group) * p.page_size + row) * D; };
    const bool whole = p.page_size % KPT == 0;   // no transfer's keys lie in two pages
    // piece tid + j NT of a stage's keys, or values: what of a transfer this lane fetches, counted from the transfer's first key
    uint32_t offset[PER_T];
    int at_key[PER_T], next_page[PER_T];
#pragma unroll
    for (int j = 0; j < PER_T; ++j) {
        const int key = (tid + j * NT) / Tile::PIECES, piece = (tid + j * NT) % Tile::PIECES ^ Tile::place(key);
        offset[j] = (uint32_t)(((whole ? lane / Tile::PIECES : 0) * D + piece * E) * sizeof(T));
        at_key[j] = whole ? __builtin_amdgcn_readfirstlane(key) : key;
    }
    auto number = [&](int stage, int j) { return std::min(stage * KT + at_key[j], p.capacity - (whole ? KPT : 1)); };   // (keys that do not exist: some that can be read)
    auto find = [&](int stage) __attribute__((always_inline)) {
        if (!whole) return;
#pragma unroll
        for (int j = 0; j < PER_T; ++j) next_page[j] = page_at(__builtin_amdgcn_readfirstlane(tree_column(p, number(stage, j))));
    };
    auto load = [&](int stage, int buffer) __attribute__((always_inline)) {
        if (whole) {
#pragma unroll
            for (int j = 0; j < PER_T; ++j) {
                const int at = number(stage, j), row = at - tree_column(p, at) * p.page_size;
                const int64_t from = row_at(next_page[j], row);
                const uint32_t to = lds0 + (uint32_t)(buffer * STAGE + (wave * WAVE + j * NT) * 16);
                attention_to_lds(K + from, offset[j], to);
                attention_to_lds(V + from, offset[j], to + HALF);
            }
        } else {
            int page[PER_T], row[PER_T];
#pragma unroll
            for (int j = 0; j < PER_T; ++j) {
                const int at = number(stage, j), column = tree_column(p, at);
                page[j] = p.table[b * p.columns + column];
                row[j] = at - column * p.page_size;
            }
            T* to = reinterpret_cast<T*>(lds + buffer * STAGE) + tid * E;
#pragma unroll
            for (int j = 0; j < PER_T; ++j) {
                const int64_t from = row_at(std::min(std::max(page[j], 0), p.pages - 1), row[j]) + offset[j] / sizeof(T);
                const Piece k = *reinterpret_cast<const Piece*>(K + from), v = *reinterpret_cast<const Piece*>(V + from);
                *reinterpret_cast<Piece*>(to + j * NT * E) = k;
                *reinterpret_cast<Piece*>(to + j * NT * E + HALF / (int)sizeof(T)) = v;
            }
        }
    };

    const uint32_t key_at = Wave::key_address(0, n, h), value_at = Wave::value_address(lane, n, h);
    f32x16 out[RB][VT];
    float base[RB], sum[RB];   // of the scores times scale_log2; the lane's share of the sum
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        base[i] = -__builtin_inff();
        sum[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < VT; ++c) out[i][c] = f32x16{};
    }

    if (count > 0) find(last - 1);
#pragma unroll
    for (int s = 0; s < NS - 1; ++s)
        if (s < count) {
            load(last - 1 - s, s);
            if (s + 1 < count) find(last - 2 - s);
        }
    int buffer = 0;
    for (int turn = 0; turn < count; ++turn, buffer = buffer + 1 == NS ? 0 : buffer + 1) {
        const int stage = last - 1 - turn;   // from the end on: a row's ancestors are met in falling order
        // the stage is in LDS, and nobody reads any more what the transfers below write
        if (turn + NS - 2 < count) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * 2 * PER_T) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
        if (turn + NS - 1 < count) {
            load(stage - (NS - 1), buffer == 0 ? NS - 1 : buffer - 1);
            if (turn + NS < count) find(stage - NS);
        }
        const uint32_t* odd = nullptr;
        if ((stage + 1) * KT > all) {
            // Keys that not all rows see: a value that is not finite must not meet the weight 0. Such values become 0 here, and the rows that see them add them below.
            T* values = reinterpret_cast<T*>(lds + buffer * STAGE + HALF);
            if (tid < KT / 32) odd_keys[(turn + 1) % 2][tid] = 0;
#pragma unroll 1
            for (int j = 0; j < PER_T; ++j) {
                const int at = tid + j * NT, key = at / Tile::PIECES;
                if (stage * KT + key < all) continue;
                Piece v = *reinterpret_cast<const Piece*>(values + at * E);
                bool finite = true;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const bool is = stage * KT + key < total && __builtin_fabsf((float)v[e]) < __builtin_inff();
                    finite &= is;
                    v[e] = is ? v[e] : (T)0.0f;
                }
                if (finite) continue;
                *reinterpret_cast<Piece*>(values + at * E) = v;
                if (stage * KT + key < total) atomicOr(&odd_keys[turn % 2][key / 32], 1u << key % 32);
            }
            __syncthreads();
            odd = odd_keys[turn % 2];
        }
#pragma unroll
        for (int u = SUB - 1; u >= 0; --u) {
            const int local = (key_wave * SUB + u) * 32, key0 = stage * KT + local;
            if (key0 >= wave_end) continue;   // (the same for the wave)
            uint32_t lds_k = lds0 + (uint32_t)(buffer * STAGE + local * Tile::ROW), lds_v = lds_k + HALF + value_at;
            lds_k += key_at;
            asm volatile("" : "+v"(lds_k), "+v"(lds_v));   // (nothing made of them is kept from one pass to the next)
            f32x16 s[RB];
            __builtin_amdgcn_s_setprio(1);
            Wave::scores(lds_k, q, s);
            __builtin_amdgcn_s_setprio(0);
            uint32_t seen[RB];   // of the 32 keys
#pragma unroll
            for (int i = 0; i < RB; ++i) seen[i] = ~0u;
            if (key0 + 32 > wave_all) {
#pragma unroll
                for (int i = 0; i < RB; ++i) {
                    if (p.parents) {
                        seen[i] = lowest_bits(length - key0);
                        while (length + ancestor[i] >= key0 && ancestor[i] >= 0) {
                            const int bit = length + ancestor[i] - key0;
                            if (bit < 32) seen[i] |= 1u << bit;
                            ancestor[i] = parents[ancestor[i]];
                        }
                    } else {
                        seen[i] = lowest_bits(length + token[i] + 1 - key0);
                    }
                    seen[i] &= lowest_bits(total - key0);
                    const uint32_t mine = seen[i] >> (4 * h);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (!(mine >> (8 * (r / 4) + r % 4) & 1)) s[i][r] = -__builtin_inff();
                }
            }
            // The base of a row's powers is the largest score so far, or up to 8 below it: P is at most 2^8, and outputs are rarely scaled. float16 has no
            // values below 2^-25 and few digits below 2^-14, where many keys of little weight may outweigh the rest: 10 to 15 below the largest score.
            constexpr float BELOW = std::is_same_v<T, f16> ? 10.0f : 0.0f, MOST = std::is_same_v<T, f16> ? 15.0f : 8.0f;
            float m[RB];
            bool far = false;
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                m[i] = s[i][0];
#pragma unroll
                for (int r = 1; r < 16; ++r) m[i] = fmaxf(m[i], s[i][r]);
                m[i] = across_halves(m[i], [](float x, float y) { return fmaxf(x, y); }) * p.scale_log2;
                far |= m[i] > base[i] + MOST;
            }
            if (__any(far)) {
#pragma unroll
                for (int i = 0; i < RB; ++i) {
                    const float now = fmaxf(base[i], m[i] - BELOW), factor = base[i] == now ? 1.0f : __builtin_amdgcn_exp2f(base[i] - now);
                    base[i] = now;
                    sum[i] *= factor;
#pragma unroll
                    for (int c = 0; c < VT; ++c) out[i][c] *= factor;
                }
            }
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                const float from = base[i] == -__builtin_inff() ? 0.0f : base[i];   // no key so far: exp2(-inf)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[i][r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], p.scale_log2, -from));
            }
            __builtin_amdgcn_s_setprio(1);
            Wave::values(lds_v, s, out, sum);
            __builtin_amdgcn_s_setprio(0);
            if (!odd) continue;
            for (uint32_t left = __builtin_amdgcn_readfirstlane(odd[local / 32]); left; left &= left - 1) {
                const int key = __builtin_ctz(left), at = key0 + key, column = tree_column(p, at);
                const T* value = V + row_at(page_at(__builtin_amdgcn_readfirstlane(column)), at - column * p.page_size);
#pragma unroll
                for (int i = 0; i < RB; ++i) {
                    float weight = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) weight = r == key / 8 * 4 + key % 4 ? s[i][r] : weight;
                    weight = __shfl(weight, n + key / 4 % 2 * 32);
                    if (!(seen[i] >> key & 1)) continue;
#pragma unroll
                    for (int c = 0; c < VT; ++c)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const float v = (float)value[32 * c + 8 * (r / 4) + 4 * h + r % 4];
                            if (!(__builtin_fabsf(v) < __builtin_inff())) out[i][c][r] += weight * v;
                        }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RB; ++i) sum[i] = across_halves(sum[i], [](float x, float y) { return x + y; });

    // ---- the shares of the keys meet, in pairs ------------------------------------------------------------
    if constexpr (KW > 1) {
        float* exchange = reinterpret_cast<float*>(lds);
        __shared__ float base_sum[KW][RW][RB][2][32];
        __syncthreads();   // nobody reads the stages any more
        if (h == 0) {
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                base_sum[key_wave][row_wave][i][0][n] = base[i];
                base_sum[key_wave][row_wave][i][1][n] = sum[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            float top = -__builtin_inff(), whole_sum = 0.0f;
#pragma unroll
            for (int w = 0; w < KW; ++w) top = fmaxf(top, base_sum[w][row_wave][i][0][n]);
            const float from = top == -__builtin_inff() ? 0.0f : top, factor = __builtin_amdgcn_exp2f(base[i] - from);
#pragma unroll
            for (int w = 0; w < KW; ++w) whole_sum = fmaf(base_sum[w][row_wave][i][1][n], __builtin_amdgcn_exp2f(base_sum[w][row_wave][i][0][n] - from), whole_sum);
            base[i] = top;
            sum[i] = whole_sum;
#pragma unroll
            for (int c = 0; c < VT; ++c) out[i][c] *= factor;
        }
#pragma unroll
        for (int step = KW / 2; step >= 1; step /= 2) {
            const int slot = (key_wave % step) * RW + row_wave;
            if (key_wave >= step && key_wave < 2 * step) {
#pragma unroll
                for (int i = 0; i < RB; ++i)
#pragma unroll
                    for (int c = 0; c < VT; ++c)
#pragma unroll
                        for (int r = 0; r < 16; ++r) exchange[(slot * RB + i) * EXCHANGE + (16 * c + r) * WAVE + lane] = out[i][c][r];
            }
            __syncthreads();
            if (key_wave < step) {
#pragma unroll
                for (int i = 0; i < RB; ++i)
#pragma unroll
                    for (int c = 0; c < VT; ++c)
#pragma unroll
                        for (int r = 0; r < 16; ++r) out[i][c][r] += exchange[(slot * RB + i) * EXCHANGE + (16 * c + r) * WAVE + lane];
            }
            __syncthreads();
        }
        if (key_wave) return;
    }

#pragma unroll
    for (int i = 0; i < RB; ++i) {
        const int64_t row = row0 + 32 * i + n;
        if (row >= rows) continue;
        if (p.splits > 1) {
            const int64_t at = (split * p.batch * p.kv_heads + slice) * rows + row;
            if (h == 0) {
                p.partial_ml[2 * at] = base[i];
                p.partial_ml[2 * at + 1] = sum[i];
            }
#pragma unroll
            for (int c = 0; c < VT; ++c)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<f32x4*>(p.partial_o + at * D + 32 * c + 8 * g + 4 * h) =
                        f32x4{out[i][c][4 * g], out[i][c][4 * g + 1], out[i][c][4 * g + 2], out[i][c][4 * g + 3]};
            continue;
        }
        const float factor = sum[i] == 0.0f ? 0.0f : 1.0f / sum[i];   // a row without keys: 0
        T* to = static_cast<T*>(p.o) + ((b * p.tokens + token[i]) * p.heads + group * p.share + (int)(row % p.share)) * D;
#pragma unroll
        for (int c = 0; c < VT; ++c)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = out[i][c][4 * g + e] * factor;
                store_values(to + 32 * c + 8 * g + 4 * h, o, 4);
            }
    }
}

// The splits of a row joined: a wave to a row, its lanes the D values.
template <class T, int D>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs p) {
    constexpr int PER_LANE = D / WAVE;
    const int64_t rows = p.tokens * p.share, all = p.batch * p.kv_heads * rows;
    const int lane = threadIdx.x % WAVE;
    const int64_t at = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;   // of a slice's row
    if (at >= all) return;
    float top = -__builtin_inff(), sum = 0.0f, o[PER_LANE] = {};
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.partial_ml[2 * (s * all + at)]);
    const float from = top == -__builtin_inff() ? 0.0f : top;
    for (int s = 0; s < p.splits; ++s) {
        const float factor = __builtin_amdgcn_exp2f(p.partial_ml[2 * (s * all + at)] - from);
        float part[PER_LANE];
        load_values(part, p.partial_o + (s * all + at) * D + lane * PER_LANE, PER_LANE);
        sum = fmaf(p.partial_ml[2 * (s * all + at) + 1], factor, sum);
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) o[e] = fmaf(part[e], factor, o[e]);
    }
#pragma unroll
    for (int e = 0; e < PER_LANE; ++e) o[e] *= sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t slice = at / rows, row = at % rows, b = slice / p.kv_heads;
    const int head = (int)(slice % p.kv_heads) * p.share + (int)(row % p.share);
    store_values(static_cast<T*>(p.o) + ((b * p.tokens + row / p.share) * p.heads + head) * D + lane * PER_LANE, o, PER_LANE);
}

enum { TREE_FEW, TREE_MID, TREE_TALL };

struct TreeCut { int form; int64_t row_blocks, workgroups, stages; };
static TreeCut tree_cut(int64_t rows, int64_t slices, int64_t keys, int bytes) {
    const int forced = tuning().tree_form;
    const int form = forced >= 0 && forced <= TREE_TALL ? forced : rows <= 32 ? TREE_FEW : rows <= 64 ? TREE_MID : TREE_TALL;
    const int64_t blocks = ceil_div(rows, (int64_t)(form == TREE_FEW ? 32 : form == TREE_MID ? 64 : 128));
    return {form, blocks, blocks * slices, ceil_div(keys, (int64_t)(form == TREE_FEW && bytes <= 256 ? 128 : 64))};
}

static int64_t tree_splits(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t size, int64_t keys, int type) {
    const int forced = tuning().tree_splits;
    if (forced > 0) return std::min(forced, 256);
    if (!batch || !tokens || !heads) return 1;
    const TreeCut cut = tree_cut(tokens * (heads / kv_heads), batch * kv_heads, keys, (int)size * (type == MI355X_TYPE_FLOAT ? 4 : 2));
    return std::max<int64_t>(1, std::min({256 / cut.workgroups, cut.stages, (int64_t)256}));
}

template <class T, int D>
static int launch_tree(TreeArgs p, hipStream_t st) {
    constexpr int BYTES = D * (int)sizeof(T);
    const int64_t rows = p.tokens * p.share, slices = p.batch * p.kv_heads;
    const TreeCut cut = tree_cut(rows, slices, p.capacity, BYTES);
    bool fits = true;
    auto launch = [&](auto rb, auto rw, auto kw, auto sub, auto ns, auto per_simd) {
        constexpr int RB = decltype(rb)::value, RW = decltype(rw)::value, KW = decltype(kw)::value, SUB = decltype(sub)::value, NS = decltype(ns)::value;
        p.row_blocks = ceil_div(rows, (int64_t)(32 * RB * RW));
        const int64_t grid = p.row_blocks * p.splits * slices;
        fits = grid_fits(grid, 64 * RW * KW) && (p.splits == 1 || grid_fits(ceil_div(slices * rows, (int64_t)4), 256));
        if (!fits) return;
        hipLaunchKernelGGL((tree_attention_kernel<T, D, RB, RW, KW, SUB, NS, decltype(per_simd)::value>), dim3((unsigned)grid), dim3(64 * RW * KW), 0, st, p);
    };
    if constexpr (BYTES <= 256) {
        if (cut.form == TREE_FEW) launch(Int<1>{}, Int<1>{}, Int<4>{}, Int<1>{}, Int<(BYTES == 128 ? 4 : 2)>{}, Int<1>{});
        else if (cut.form == TREE_MID) launch(Int<1>{}, Int<2>{}, Int<2>{}, Int<1>{}, Int<(BYTES == 128 ? 4 : 2)>{}, Int<2>{});
        else launch(Int<1>{}, Int<4>{}, Int<1>{}, Int<2>{}, Int<2>{}, Int<2>{});
    } else if constexpr (BYTES == 512) {
        if (cut.form == TREE_FEW) launch(Int<1>{}, Int<1>{}, Int<2>{}, Int<1>{}, Int<2>{}, Int<1>{});
        else if (cut.form == TREE_MID) launch(Int<1>{}, Int<2>{}, Int<2>{}, Int<1>{}, Int<2>{}, Int<1>{});
        else launch(Int<1>{}, Int<4>{}, Int<1>{}, Int<1>{}, Int<2>{}, Int<1>{});
    } else {
        if (cut.form == TREE_FEW) launch(Int<1>{}, Int<1>{}, Int<1>{}, Int<1>{}, Int<2>{}, Int<1>{});
        else if (cut.form == TREE_MID) launch(Int<1>{}, Int<2>{}, Int<1>{}, Int<1>{}, Int<2>{}, Int<1>{});
        else launch(Int<1>{}, Int<4>{}, Int<1>{}, Int<1>{}, Int<2>{}, Int<1>{});
    }
    MI355X_REQUIRE(fits, "tree_attention: too large");
    if (p.splits > 1) hipLaunchKernelGGL((tree_join_kernel<T, D>), dim3((unsigned)ceil_div(slices * rows, (int64_t)4)), dim3(256), 0, st, p);
    return check_launch("tree_attention_kernel");
}

static bool tree_fits(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t size, int64_t page_size, int64_t columns) {
    return batch >= 0 && tokens >= 0 && heads >= 0 && heads < 1 << 20 && kv_heads >= 1 && heads % kv_heads == 0 && (size == 64 || size == 128 || size == 256) && page_size >= 1 &&
           columns >= 0 && batch < (int64_t)1 << 31 && tokens < (int64_t)1 << 31 && page_size < (int64_t)1 << 31 && columns < (int64_t)1 << 31 &&
           page_size * columns < ((int64_t)1 << 31) - 1024 && (double)batch * tokens * heads < 0x1p40;
}

}  // namespace mi355x

extern "C" int64_t mi355x_tree_attention_scratch(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t size, int64_t page_size, int64_t columns, int type) {
    using namespace mi355x;
    if (!is_mixed_type(type) || !tree_fits(batch, tokens, heads, kv_heads, size, page_size, columns)) return 0;
    const int64_t splits = tree_splits(batch, tokens, heads, kv_heads, size, page_size * columns, type);
    return splits > 1 ? splits * batch * tokens * heads * (size + 2) : 0;
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
    const int64_t splits = tree_splits(batch, tokens, heads, kv_heads, size, page_size * columns, type), floats = splits > 1 ? splits * batch * tokens * heads * (size + 2) : 0;
    MI355X_REQUIRE(floats == 0 || (scratch && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0 && scratch_floats >= floats), "tree_attention: scratch memory for %lld floats, 16-byte aligned",
                   (long long)floats);
    TreeArgs p = {};
    p.q = Q; p.k_pages = k_pages; p.v_pages = v_pages; p.table = table; p.lengths = lengths; p.parents = parents; p.o = O;
    p.partial_o = scratch;
    p.partial_ml = scratch ? scratch + splits * batch * tokens * heads * size : nullptr;
    p.batch = batch; p.tokens = tokens; p.columns = columns;
    p.pages = (int)pages; p.page_size = (int)page_size; p.capacity = (int)(page_size * columns);
    p.heads = (int)heads; p.kv_heads = (int)kv_heads; p.share = (int)(heads / kv_heads); p.splits = (int)splits;
    while (((int64_t)1 << p.page_shift) < page_size) ++p.page_shift;
    p.page_magic = (uint32_t)((((uint64_t)1 << (31 + p.page_shift)) + (uint64_t)page_size - 1) / (uint64_t)page_size);
    p.scale_log2 = scale * 1.44269504088896340736f;
    int status = MI355X_OK;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        hipStream_t st = static_cast<hipStream_t>(stream);
        status = size == 64 ? launch_tree<T, 64>(p, st) : size == 128 ? launch_tree<T, 128>(p, st) : launch_tree<T, 256>(p, st);
    });
    return status;
}
