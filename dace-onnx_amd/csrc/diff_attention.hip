// DifferentialAttention: O = (softmax(c Q1 K1^T) - l softmax(c Q2 K2^T)) V with l = exp(q1 . k1) - exp(q2 . k2) + l0 from learned vectors. The two maps of
// a head have queries and keys of their own, d values each, and share values of 2 d; H / G heads share keys and values. Arrays in float32, float16 or
// bfloat16; scores, running maxima, sums and outputs in float32. The reference has no such node.
//
// One pass over the keys with a running maximum and sum, as two attentions that read the same values: a wave has one map of RB blocks of 32 rows (a
// row: one query of one of the heads that share keys), its neighbour the other map, and at the end one takes the other's output from its own.
//   * S^T = K Q^T by 32 x 32 MFMA tiles: lane (n, h) gets 16 scores of row n, of the keys 8 (r / 4) + 4 h + r % 4. Largest score and sum of a row are
//     15 steps in the lane and one across lanes n and n + 32.
//   * Those registers are the second product's operand as they stand: O^T = V^T P^T, whose k indices are dealt to the lanes the same way. With 16-bit
//     values V's operand comes from LDS by transposing reads, with float32 by 4-byte reads (and is split in three, see Operand). Every lane has one row: a running maximum that
//     changes is one factor to a lane.
//   * Keys and values are staged through LDS for all waves, 16-byte pieces permuted within a row so that reads of a column meet no bank twice.
// P is rounded to the arrays' type for the second product, half a step of it, because the matrix unit takes it in no more than 16 bits at the rate of that type (errors of
// bfloat16 results in the 2-norm 1.7e-3 to 2.0e-3, where rounding the results alone gives 1.7e-3); the sum is that of the rounded values, so that the weights add up to one.
// Few rows: the keys are dealt to `splits` workgroups, whose maxima, sums and outputs a second launch joins.
// Bound by matrix and vector instructions one after the other (a vector instruction takes its time from the matrix pipe): 768 cycles of products and about 1000 of exponentials,
// maxima and roundings for 32 keys, 64 rows and a map of 64. 8 heads of 64 over 8192 queries and keys in bfloat16: 382 us, 1.08 PFLOP/s of the 12 d operations that one
// pass with two outputs takes for a pair, where a library product of 8192^3 reaches 1.15 to 1.51; causal 228. Two waves to a SIMD have 256
// registers each, most of them accumulators: what else is kept from pass to pass decides whether those stay in place. float32: 3 x 333 queries and keys, 6 heads of 64, 21 us; 8 x 3 heads, 4016 x 6818: 2.8 ms, 180
// TFLOP/s (float32 products reach 154). Few rows by the bytes: 8 x 1 of up to 8192 keys, 90 MB, 20 us (4.5 TB/s) and 4 for the second launch.
#include "attention_tile.h"
#include "gemm_tile.h"

#include <algorithm>

namespace mi355x {

struct DiffArgs {
    const void* Q; const void* K; const void* V; void* O;
    const float* q1; const float* k1; const float* q2; const float* k2;
    const int32_t* lengths;
    float* partial_o; float* partial_ml;   // of splits; [split][slice][row][map][2 d], [split][slice][row][map][2]
    int64_t batch, Sq, Sk;
    int heads, groups, share, vector;   // share = heads / groups; vector: length of the learned vectors
    int causal, splits;
    int64_t row_blocks;                 // of the rows Sq * share of a slice (one batch entry, one group)
    int per_xcd;                        // slices of an XCD whose blocks take turns; 0: one slice after the other; -1: all slices take turns
    float scale_log2, lambda_init;
};

__device__ __forceinline__ float diff_lambda(const DiffArgs& p) {
    float a = 0.0f, b = 0.0f;
    for (int i = threadIdx.x % WAVE; i < p.vector; i += WAVE) {
        a = fmaf(p.q1[i], p.k1[i], a);
        b = fmaf(p.q2[i], p.k2[i], b);
    }
    return expf(wave_sum(a)) - expf(wave_sum(b)) + p.lambda_init;
}

// keys that batch entry b has; what a caller wrote beyond the array is taken as all of it
__device__ __forceinline__ int64_t diff_length(const DiffArgs& p, int64_t b) {
    if (!p.lengths) return p.Sk;
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : n > p.Sk ? p.Sk : n;
}

// Waves: two maps, RW blocks of 32 RB rows, KW shares of a stage's keys, 32 SUB each. Two stages: while one is multiplied the other is on its way. DIRECT: by
// transfers that need no registers (arrays at 16-byte boundaries); the last stage, whose missing keys have to be zeros, always goes through registers, and
// so do all stages of arrays at other addresses.
template <class T, int D, int RB, int RW, int KW, int SUB, bool DIRECT>
__global__ __launch_bounds__(128 * RW * KW, 2) void diff_attention_kernel(DiffArgs p) {
    using Tile = AttentionTile<T, 2 * D>;
    using Wave = AttentionWave<T, 2 * D, D>;
    using Piece = typename Wave::Piece;
    using UnalignedPiece = typename Wave::UnalignedPiece;
    constexpr int KT = 32 * KW * SUB, E = Tile::E, NT = 128 * RW * KW, VT = Wave::VT, ROWS = 32 * RB * RW;
    constexpr int HALF = KT * Tile::ROW, STAGE = 2 * HALF;            // keys, then values
    constexpr int PER_T = KT * Tile::PIECES / NT;
    static_assert(KT * Tile::PIECES % NT == 0 && Tile::PIECES <= WAVE, "whole pieces to a thread, whole rows to a transfer");
    constexpr int EXCHANGE = 32 * 2 * D;   // floats of a row block's output
    __shared__ __attribute__((aligned(1024))) unsigned char lds[std::max(2 * STAGE, 4 * EXCHANGE * (KW == 1 ? RW : KW * RW * RB))];

    const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int n = lane % 32, h = lane / 32, map = wave % 2, row_wave = wave / 2 % RW, key_wave = wave / (2 * RW);
    const int64_t logical = xcd_remap(blockIdx.x, (int64_t)gridDim.x);
    int64_t turn, slice;
    int split = 0;
    if (p.per_xcd < 0) {
        const int64_t slices = p.batch * p.groups;
        turn = blockIdx.x / slices;
        slice = blockIdx.x % slices;
    } else if (p.per_xcd) {
        const int64_t each = p.row_blocks * p.per_xcd, local = logical % each;
        turn = local / p.per_xcd;
        slice = logical / each * p.per_xcd + local % p.per_xcd;
    } else {
        const int64_t rest = logical / p.row_blocks;
        turn = logical % p.row_blocks;
        split = (int)(rest % p.splits);
        slice = rest / p.splits;
    }
    const int64_t b = slice / p.groups;
    const int group = (int)(slice % p.groups);
    const int64_t rows = p.Sq * p.share, length = diff_length(p, b);
    const int64_t ahead = length - p.Sq;   // if causal, query i sees the keys up to i + ahead
    auto keys_of = [&](int64_t row) { return p.causal ? std::max((int64_t)0, std::min(length, row / p.share + ahead + 1)) : length; };

    const int64_t block = p.causal ? p.row_blocks - 1 - turn : turn;   // long ones first

    // ---- queries: row r of a slice is head r % share of query r / share ------------------------------------
    const int64_t row0 = block * ROWS + row_wave * RB * 32;   // of the wave
    int seen[RB];   // keys of the row
    Operand<T> q[RB][Wave::QP];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        const int64_t row = row0 + 32 * i + n, r = row < rows ? row : rows - 1, query = r / p.share;
        const int head = group * p.share + (int)(r % p.share);
        seen[i] = (int)keys_of(r);
        const T* from = static_cast<const T*>(p.Q) + ((b * p.Sq + query) * 2 * p.heads + 2 * head + map) * D + 8 * h;
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
    // keys that any row of the workgroup sees; that any row of the wave sees, and that all of its rows see
    const int end = (int)keys_of(std::min(rows, (block + 1) * ROWS) - 1);
    const int wave_end = __builtin_amdgcn_readfirstlane((int)keys_of(std::min(rows, row0 + 32 * RB) - 1));
    const int wave_all = __builtin_amdgcn_readfirstlane((int)keys_of(std::min(rows - 1, row0)));
    const int stages = (end + KT - 1) / KT, per_split = (stages + p.splits - 1) / p.splits;
    const int first = split * per_split, last = std::min(stages, first + per_split);

    const T* K = static_cast<const T*>(p.K) + (b * p.Sk * p.groups + group) * 2 * D;
    const T* V = static_cast<const T*>(p.V) + (b * p.Sk * p.groups + group) * 2 * D;
    const int64_t key_stride = (int64_t)p.groups * 2 * D;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds;

    // piece tid + j NT of a stage's keys, or values: where it is in memory and, of a transfer, what of it this lane fetches
    uint32_t offset[DIRECT ? PER_T : 1];
    if constexpr (DIRECT) {
#pragma unroll
        for (int j = 0; j < PER_T; ++j) {
            const int key = (tid + j * NT) / Tile::PIECES, piece = (tid + j * NT) % Tile::PIECES ^ Tile::place(key);
            offset[j] = (uint32_t)((key * key_stride + piece * E) * sizeof(T));
        }
    }
    auto by_registers = [&](int stage, int buffer) __attribute__((always_inline)) {
        constexpr int BATCH = PER_T < 4 ? PER_T : 4;
        T* to = reinterpret_cast<T*>(lds + buffer * STAGE);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll 1
            for (int j0 = 0; j0 < PER_T; j0 += BATCH) {
                Piece held[BATCH];
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const int at = tid + (j0 + j) * NT, piece = at % Tile::PIECES, key = at / Tile::PIECES;
                    held[j] = Piece{};
                    if (stage * (int64_t)KT + key < length)   // (keys that do not exist may lie outside, or hold anything)
                        held[j] = *reinterpret_cast<const UnalignedPiece*>((half ? V : K) + (stage * (int64_t)KT + key) * key_stride + piece * E);
                }
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const int at = tid + (j0 + j) * NT, piece = at % Tile::PIECES, key = at / Tile::PIECES;
                    *reinterpret_cast<Piece*>(to + half * (HALF / (int)sizeof(T)) + Tile::at(key, piece)) = held[j];
                }
            }
    };
    auto load = [&](int stage, int buffer) __attribute__((always_inline)) {
        if constexpr (DIRECT) {
            if ((stage + 1) * (int64_t)KT <= length) {
                const int64_t at = stage * (int64_t)KT * key_stride;
#pragma unroll
                for (int j = 0; j < PER_T; ++j) {
                    const uint32_t to = lds0 + (uint32_t)(buffer * STAGE + (wave * WAVE + j * NT) * 16);
                    attention_to_lds(K + at, offset[j], to);
                    attention_to_lds(V + at, offset[j], to + HALF);
                }
                return;
            }
        }
        by_registers(stage, buffer);
    };

    const uint32_t key_at = Wave::key_address(map, n, h), value_at = Wave::value_address(lane, n, h);
    f32x16 out[RB][VT];
    float base[RB], sum[RB];   // of the scores times scale_log2; the lane's share of the sum
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        base[i] = -__builtin_inff();
        sum[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < VT; ++c) out[i][c] = f32x16{};
    }

    static_assert(PER_T % (PER_T < 4 ? PER_T : 4) == 0, "whole batches");
    if (first < last) load(first, 0);
    for (int stage = first, buffer = 0; stage < last; ++stage, buffer ^= 1) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // the stage is in LDS, and nobody reads the other one any more
        __syncthreads();
        if (stage + 1 < last) load(stage + 1, buffer ^ 1);
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const int local = (key_wave * SUB + u) * 32, key0 = stage * KT + local;
            if (key0 >= wave_end) break;   // (the same for the wave)
            uint32_t lds_k = lds0 + (uint32_t)(buffer * STAGE + local * Tile::ROW), lds_v = lds_k + HALF + value_at;
            lds_k += key_at;
            asm volatile("" : "+v"(lds_k), "+v"(lds_v));   // (nothing made of them is kept from one pass to the next)
            f32x16 s[RB];
            __builtin_amdgcn_s_setprio(1);
            Wave::scores(lds_k, q, s);
            __builtin_amdgcn_s_setprio(0);
            if (key0 + 32 > wave_all) {
#pragma unroll
                for (int i = 0; i < RB; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (key0 + 8 * (r / 4) + 4 * h + r % 4 >= seen[i]) s[i][r] = -__builtin_inff();
            }
            // The base of a row's powers is the largest score so far, or up to 8 below it: P is at most 2^8, and outputs are rarely scaled. float16 has no
            // values below 2^-25 and few digits below 2^-14, where many keys of little weight may outweigh the rest: 10 to 15 below the largest score: 12 would cost 2 to 5 %.
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
        }
    }
#pragma unroll
    for (int i = 0; i < RB; ++i) sum[i] = across_halves(sum[i], [](float x, float y) { return x + y; });

    // ---- the shares of the keys meet, in pairs ------------------------------------------------------------
    float* exchange = reinterpret_cast<float*>(lds);
    if constexpr (KW > 1) {
        __shared__ float base_sum[KW][RW][2][RB][2][32];
        __syncthreads();   // nobody reads the stages any more
        if (h == 0) {
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                base_sum[key_wave][row_wave][map][i][0][n] = base[i];
                base_sum[key_wave][row_wave][map][i][1][n] = sum[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            float top = -__builtin_inff(), total = 0.0f;
#pragma unroll
            for (int w = 0; w < KW; ++w) top = fmaxf(top, base_sum[w][row_wave][map][i][0][n]);
            const float from = top == -__builtin_inff() ? 0.0f : top, factor = __builtin_amdgcn_exp2f(base[i] - from);
#pragma unroll
            for (int w = 0; w < KW; ++w) total = fmaf(base_sum[w][row_wave][map][i][1][n], __builtin_amdgcn_exp2f(base_sum[w][row_wave][map][i][0][n] - from), total);
            base[i] = top;
            sum[i] = total;
#pragma unroll
            for (int c = 0; c < VT; ++c) out[i][c] *= factor;
        }
#pragma unroll
        for (int step = KW / 2; step >= 1; step /= 2) {
            const int slot = ((key_wave % step) * RW + row_wave) * 2 + map;
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
    }

    // ---- the two maps meet --------------------------------------------------------------------------------
    const bool result = key_wave == 0;
    const float weight = p.splits > 1 ? 0.0f : diff_lambda(p);
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        const int64_t row = row0 + 32 * i + n;
        if (p.splits > 1) {
            if (result && row < rows) {
                const int64_t at = ((split * p.batch * p.groups + slice) * rows + row) * 2 + map;
                if (h == 0) {
                    p.partial_ml[2 * at] = base[i];
                    p.partial_ml[2 * at + 1] = sum[i];
                }
#pragma unroll
                for (int c = 0; c < VT; ++c)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<f32x4*>(p.partial_o + at * 2 * D + 32 * c + 8 * g + 4 * h) =
                            f32x4{out[i][c][4 * g], out[i][c][4 * g + 1], out[i][c][4 * g + 2], out[i][c][4 * g + 3]};
            }
            continue;
        }
        const float factor = sum[i] == 0.0f ? 0.0f : (map ? weight : 1.0f) / sum[i];   // a row without keys: 0
        float* other = exchange + row_wave * EXCHANGE;
        __syncthreads();
        if (result && map == 1) {
#pragma unroll
            for (int c = 0; c < VT; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) other[(16 * c + r) * WAVE + lane] = out[i][c][r] * factor;
        }
        __syncthreads();
        if (result && map == 0 && row < rows) {
            const int64_t query = row / p.share;
            const int head = group * p.share + (int)(row % p.share);
            T* to = static_cast<T*>(p.O) + ((b * p.Sq + query) * p.heads + head) * 2 * D;
#pragma unroll
            for (int c = 0; c < VT; ++c)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = out[i][c][4 * g + e] * factor - other[(16 * c + 4 * g + e) * WAVE + lane];
                    store_values(to + 32 * c + 8 * g + 4 * h, o, 4);
                }
        }
    }
}

// The splits of a row joined: a wave to a row and map, its lanes the 2 D values, its first BATCH
// reads on their way before anything is needed.
template <class T, int D, int BATCH>
__global__ __launch_bounds__(256) void diff_join_kernel(DiffArgs p) {
    constexpr int PER_LANE = 2 * D / WAVE;
    __shared__ float other[2][2 * D];
    const int64_t rows = p.Sq * p.share, all = p.batch * p.groups * rows;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), map = wave % 2;
    int64_t at = (int64_t)blockIdx.x * 2 + wave / 2;   // of a slice's row
    const bool mine = at < all;
    if (!mine) at = all - 1;
    // lane s has the base and the sum of splits s, s + 64, ...
    float base[4], sums[4], top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int s = lane + i * WAVE;
        const bool is = s < p.splits;
        base[i] = is ? p.partial_ml[2 * ((s * all + at) * 2 + map)] : -__builtin_inff();
        sums[i] = is ? p.partial_ml[2 * ((s * all + at) * 2 + map) + 1] : 0.0f;
    }
    const float* from_split = p.partial_o + (at * 2 + map) * 2 * D + lane * PER_LANE;
    float part[BATCH][PER_LANE];
    auto fetch = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) load_values(part[j], from_split + (s0 + j < p.splits ? s0 + j : p.splits - 1) * all * 4 * D, PER_LANE);
    };
    fetch(0);
    const float weight = map ? diff_lambda(p) : 1.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, base[i]);
    top = wave_max(top);
    const float from = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        base[i] = __builtin_amdgcn_exp2f(base[i] - from);
        sum = fmaf(sums[i], base[i], sum);
    }
    sum = wave_sum(sum);
    float o[PER_LANE] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int count = p.splits - i * WAVE < WAVE ? p.splits - i * WAVE : WAVE;
        for (int s0 = 0; s0 < count; s0 += BATCH) {
            if (i || s0) fetch(i * WAVE + s0);
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const bool is = s0 + j < count;
                const float factor = is ? readlane_f32(base[i], s0 + j) : 0.0f;
#pragma unroll
                for (int e = 0; e < PER_LANE; ++e) o[e] = fmaf(is ? part[j][e] : 0.0f, factor, o[e]);
            }
        }
    }
    const float factor = sum == 0.0f ? 0.0f : weight / sum;
    if (map) {
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) other[wave / 2][lane * PER_LANE + e] = o[e] * factor;
    }
    __syncthreads();
    if (map || !mine) return;
#pragma unroll
    for (int e = 0; e < PER_LANE; ++e) o[e] = o[e] * factor - other[wave / 2][lane * PER_LANE + e];
    const int64_t slice = at / rows, row = at % rows, b = slice / p.groups;
    const int head = (int)(slice % p.groups) * p.share + (int)(row % p.share);
    store_values(static_cast<T*>(p.O) + ((b * p.Sq + row / p.share) * p.heads + head) * 2 * D + lane * PER_LANE, o, PER_LANE);
}

// How a type and head size are cut: with many rows RW x RB blocks of 32 and SUB blocks of 32 keys in a stage; with few rows one block and KW key waves.
template <class T, int D>
struct DiffForm {
    static constexpr int BYTES = D * (int)sizeof(T);   // 64 to 512
    static constexpr int RB = BYTES <= 128 ? 2 : 1, RW = 2, SUB = BYTES <= 128 ? 2 : 1;
    static constexpr int KW = BYTES <= 128 ? 4 : BYTES <= 256 ? 2 : 1, WIDE = BYTES <= 256 ? 2 : 1;
};

// Which form. FEW: one block of rows and KW key waves to a workgroup, one workgroup to a CU; SMALL: half the key waves, two to a CU (small heads); WIDE: many rows by
// two key waves, one to a CU, where the long and short blocks of a causal mask even out; TALL: by one, two to a CU. Microseconds FEW / SMALL / WIDE / TALL, bfloat16,
// 8 heads of 64: 512 queries and keys 11.0 / 11.8 / 20.7 / 21.7; 1039 (264 blocks of rows) 34 / 23 / 35 / 41; 1500 41 / 30 / 45 / 55; 2048 49 / - / 54 / 68; 8192 699 / - /
// 441 / 394. Heads of 128, 1039: 75 / 59 / 40 / 50; in three parts 1200 of 4000, 4 heads 97 / - / 59 / 72 (one part 121 / - / 112 / 162). float32, heads of 64: 3 x 333 24.8 / - /
// 29.9 / 32.8, 1039 117 / 102 / 79 / 93.
enum { DIFF_FEW, DIFF_TALL, DIFF_WIDE, DIFF_SMALL };

// Of a causal mask, heads of at most 128 bytes: a form's time is that of the longest block, of all blocks, or, where there are more workgroups than places, of the two that
// follow one another; long ones start first. `row`: us for a key and 32 rows where all places are taken, `block`: for a key and a workgroup, `start`: for each round.
// 4 heads of 64, bfloat16: 4000 56 / 68 / 103; 8 heads: 1200 19.0 / 22.0 / 35.5, 2048 35.0 / 34.9 / 55.6, 2600 53 / 46.8 / 71.8, 8192 348 / - / 232; 4 x 600 26.6 / 15.9 / 25.4;
// float32, heads of 32: 2 x 1644 86 / 74 / 104, 10 x 564 of 3435, 3 heads 215 / 214 / 200.
static int diff_causal_form(int64_t few, int64_t wide, int64_t Sq, int64_t Sk) {
    const double longest = (double)Sk, shortest = std::max(0.0, (double)(Sk - Sq)), mean = Sq <= Sk ? longest - 0.5 * (double)Sq : 0.5 * longest * longest / (double)Sq;
    auto cost = [&](int64_t workgroups, int64_t places, double row, double block, double start) {
        double most = std::max(longest * block, (double)few * mean * row / 256.0);
        if (workgroups > places) most = std::max(most, 2.0 * block * (longest - (longest - shortest) * (double)places / (double)workgroups));
        return most + start * (double)workgroups / (double)places;
    };
    const double as_few = cost(few, 256, 0.0102, 0.0102, 4.0), as_small = cost(few, 512, 0.0078, 0.0156, 2.0), as_wide = cost(wide, 256, 0.0067, 0.0269, 2.0);
    return as_few <= as_small && as_few <= as_wide ? DIFF_FEW : as_small <= as_wide ? DIFF_SMALL : DIFF_WIDE;
}

struct DiffCut { int form; int64_t workgroups, stages; };
static DiffCut diff_cut(int64_t rows, int64_t slices, int64_t Sq, int64_t Sk, int bytes, int causal, bool in_parts) {
    const int forced = tuning().diff_form;
    const int64_t few = ceil_div(rows, (int64_t)32) * slices, wide = ceil_div(rows, (int64_t)(bytes <= 128 ? 128 : 64)) * slices;
    const int form = forced >= 0 && forced <= DIFF_SMALL ? forced :
                     in_parts && bytes <= 128 && rows <= 32 ? DIFF_SMALL :
                     in_parts && bytes == 256 && few > 128 ? DIFF_WIDE :   // (FEW has no room for parts)
                     rows <= 32 || (few <= 256 && bytes <= 256) ? DIFF_FEW :
                     causal && bytes <= 128 && !in_parts ? diff_causal_form(few, wide, Sq, Sk) :
                     few <= 512 && bytes <= 128 ? DIFF_SMALL :
                     causal || wide <= 256 ? DIFF_WIDE : DIFF_TALL;
    const bool one_block = form == DIFF_FEW || form == DIFF_SMALL;
    const int64_t keys = bytes > 256 ? 32 : form == DIFF_FEW && bytes <= 128 ? 128 : form == DIFF_SMALL && bytes > 128 ? 32 : 64;
    return {form, one_block ? few : wide, ceil_div(Sk, keys)};
}

template <class T, int D>
static int launch_diff(DiffArgs p, hipStream_t st) {
    using F = DiffForm<T, D>;
    const int64_t rows = p.Sq * p.share, slices = p.batch * p.groups;
    const bool direct = ((reinterpret_cast<uintptr_t>(p.K) | reinterpret_cast<uintptr_t>(p.V)) & 15) == 0 && (int64_t)p.groups * D < 1 << 20;
    bool fits = true;
    auto launch = [&](auto rb, auto rw, auto kw, auto sub) {
        constexpr int RB = decltype(rb)::value, RW = decltype(rw)::value, KW = decltype(kw)::value, SUB = decltype(sub)::value;
        p.row_blocks = ceil_div(rows, (int64_t)(32 * RB * RW));
        const int64_t grid = p.row_blocks * p.splits * slices;
        fits = grid_fits(grid, 128 * RW * KW) && (p.splits == 1 || grid_fits(ceil_div(slices * rows, (int64_t)2), 256));
        if (!fits) return;
        // long blocks of a causal mask first, whichever slice they are of: of the slices whose keys an XCD's L2 holds, or of all
        p.per_xcd = !p.causal || p.splits > 1 ? 0 : slices % NUM_XCD == 0 ? (int)(slices / NUM_XCD) : -1;
        const dim3 g((unsigned)grid), block(128 * RW * KW);
        if (direct) hipLaunchKernelGGL((diff_attention_kernel<T, D, RB, RW, KW, SUB, true>), g, block, 0, st, p);
        else hipLaunchKernelGGL((diff_attention_kernel<T, D, RB, RW, KW, SUB, false>), g, block, 0, st, p);
    };
    const int form = diff_cut(rows, slices, p.Sq, p.Sk, F::BYTES, p.causal, p.splits > 1).form;
    if (form == DIFF_FEW) launch(Int<1>{}, Int<1>{}, Int<F::KW>{}, Int<1>{});
    else if (form == DIFF_SMALL) launch(Int<1>{}, Int<1>{}, Int<(F::KW > 1 ? F::KW / 2 : 1)>{}, Int<1>{});
    else if (form == DIFF_WIDE) launch(Int<F::RB>{}, Int<F::RW>{}, Int<F::WIDE>{}, Int<1>{});
    else launch(Int<F::RB>{}, Int<F::RW>{}, Int<1>{}, Int<F::SUB>{});
    MI355X_REQUIRE(fits, "differential_attention: too large");
    if (p.splits > 1) {
        // (2 parts of 8192 rows by sixteen reads 4 us more than by four)
        const dim3 g((unsigned)ceil_div(slices * rows, (int64_t)2));
        if (p.splits <= 4) hipLaunchKernelGGL((diff_join_kernel<T, D, 4>), g, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((diff_join_kernel<T, D, 16>), g, dim3(256), 0, st, p);
    }
    return check_launch("diff_attention_kernel");
}

// whether products of them fit 64 bits, and keys with the stage that they end in 32
static bool diff_fits(int64_t batch, int64_t Sq, int64_t Sk, int64_t heads, int64_t groups) {
    return Sq < (int64_t)1 << 31 && Sk < ((int64_t)1 << 31) - 256 && heads < 1 << 20 && batch < (int64_t)1 << 31 && (double)batch * Sq * heads < 0x1p40 &&
           (double)batch * Sk * groups < 0x1p40;
}

}  // namespace mi355x

extern "C" int64_t mi355x_differential_attention_splits(int64_t batch, int64_t Sq, int64_t Sk, int64_t heads, int64_t groups, int64_t size, int type) {
    using namespace mi355x;
    if (!is_mixed_type(type) || (size != 32 && size != 64 && size != 128) || groups < 1 || heads < 1 || heads % groups || batch < 1 || Sq < 1 || Sk < 1 || !diff_fits(batch, Sq, Sk, heads, groups)) return 1;
    const int64_t rows = Sq * (heads / groups), slices = batch * groups;
    const int bytes = (int)size * (type == MI355X_TYPE_FLOAT ? 4 : 2);
    const DiffCut whole = diff_cut(rows, slices, Sq, Sk, bytes, 0, false), part = diff_cut(rows, slices, Sq, Sk, bytes, 0, true);
    const int forced = tuning().diff_splits;
    if (forced > 0) return std::min(forced, 256);
    // A causal call is priced as one without a mask: every row as if it saw all keys, and of one part the form that the call would take without the mask.
    // By what a workgroup's stages take, what joining takes (a launch, and the sums written and read), and one round of workgroups at most. Measured, microseconds: 8 x 1 of
    // 8192 keys, 16 heads in 4 groups, 64, bfloat16: 100 in one part (FEW), 32 in 8, 28 in 16, 32 in 32 (SMALL); 1 x 1 of them 16.1 in 16, 13.0 in 32; 16 x 1 of 1000 keys, 8 heads,
    // float16: 20.6 in one part, 19.7 in 2, 17.7 in 4; 512 of 512, 8 heads: 11.3 and 18.2; float32: 333 of 333, 6 heads of 64, 24.8 in one part, 21.7 in 2, 19.5 in 3; 8 heads
    // of 128, 1024 of 1024: 162 and 109, 256 of 256 47, 36, 31.6 in 4; 2 heads, 2228 of 2228: of 64, float32 119 and 71 in 3 (WIDE), of 128, bfloat16, causal 72 and 42.5, 3344 of 3344 101
    // and 66 in 2.
    auto stage = [&](const DiffCut& c) { 
        const bool wide = c.form == DIFF_WIDE || c.form == DIFF_TALL;   // us
        return type == MI355X_TYPE_FLOAT ? (size == 128 ? 4.5 : size == 64 ? (wide ? 4.2 : 3.2) : 2.3) : size == 128 ? (wide ? 1.8 : 1.9) : c.form == DIFF_SMALL ? 1.0 : 1.3;
    };
    const double sums = 16.0 * (double)(batch * Sq * heads) * (double)(2 * size + 2) / 4e6;                                                  // of one part
    const int64_t room = (part.form == DIFF_SMALL ? 512 : 256) / part.workgroups;
    int64_t best = 1;
    double least = stage(whole) * (double)whole.stages;
    for (int64_t n = 2; n <= std::min({room, part.stages, (int64_t)256}); ++n) {
        const double cost = stage(part) * (double)ceil_div(part.stages, n) + 4.0 + (double)n * (0.1 + sums);
        if (cost < least) least = cost, best = n;
    }
    return best;
}

extern "C" int mi355x_differential_attention(const void* Q, const void* K, const void* V, const float* lambda_q1, const float* lambda_k1,
                                             const float* lambda_q2, const float* lambda_k2, const int32_t* lengths, void* O, float* scratch,
                                             int64_t batch, int64_t Sq, int64_t Sk, int64_t heads, int64_t groups, int64_t size, int64_t vector,
                                             float lambda_init, float scale, int causal, int64_t splits, int type, void* stream) {
    using namespace mi355x;
    MI355X_REQUIRE(batch >= 0 && Sq >= 0 && Sk >= 0 && heads >= 0 && vector >= 0, "differential_attention: negative extent");
    MI355X_REQUIRE(is_mixed_type(type), "differential_attention: element type %d", type);
    MI355X_REQUIRE(size == 32 || size == 64 || size == 128, "differential_attention: head size %lld (32, 64 and 128 are supported)", (long long)size);
    MI355X_REQUIRE(groups >= 1 && heads % groups == 0, "differential_attention: %lld heads share keys and values in %lld groups", (long long)heads, (long long)groups);
    MI355X_REQUIRE(scale > 0.0f && scale < __builtin_inff(), "differential_attention: scale %g (a positive number is needed)", (double)scale);
    MI355X_REQUIRE(splits >= 1 && splits <= 256, "differential_attention: %lld splits (1 to 256)", (long long)splits);
    if (batch == 0 || Sq == 0 || heads == 0) return MI355X_OK;
    MI355X_REQUIRE(Q && O && (Sk == 0 || (K && V)) && (vector == 0 || (lambda_q1 && lambda_k1 && lambda_q2 && lambda_k2)), "differential_attention: null pointer");
    MI355X_REQUIRE(splits == 1 || (scratch && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0), "differential_attention: splits need scratch memory, 16-byte aligned");
    MI355X_REQUIRE(diff_fits(batch, Sq, Sk, heads, groups) && vector < 1 << 20, "differential_attention: too large");
    DiffArgs p = {};
    p.Q = Q; p.K = K; p.V = V; p.O = O; p.q1 = lambda_q1; p.k1 = lambda_k1; p.q2 = lambda_q2; p.k2 = lambda_k2; p.lengths = lengths;
    p.batch = batch; p.Sq = Sq; p.Sk = Sk; p.heads = (int)heads; p.groups = (int)groups; p.share = (int)(heads / groups); p.vector = (int)vector;
    p.causal = causal != 0; p.splits = (int)splits;
    p.partial_o = scratch;
    p.partial_ml = scratch ? scratch + splits * batch * heads * Sq * 2 * 2 * size : nullptr;
    p.scale_log2 = scale * 1.44269504088896340736f;
    p.lambda_init = lambda_init;
    int status = MI355X_OK;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        hipStream_t st = static_cast<hipStream_t>(stream);
        status = size == 32 ? launch_diff<T, 32>(p, st) : size == 64 ? launch_diff<T, 64>(p, st) : launch_diff<T, 128>(p, st);
    });
    return status;
}
