// DifferentialAttention: O = (softmax(c Q1 K1^T) - l softmax(c Q2 K2^T)) V with l = exp(q1 . k1) - exp(q2 . k2) + l0 from learned vectors. The two maps of
// a head have queries and keys of their own, d values each, and share values of 2 d; H / G heads share keys and values. Arrays in float32, float16 or
// bfloat16; scores, running maxima, sums and outputs in float32. The reference has no such node.
//
// One pass over the keys with a running maximum and sum, as two attentions that read the same values: a wave has one map of RB blocks of 32 rows (a
// row: one query of one of the heads that share keys), its neighbour the other map, and at the end one takes the other's output from its own.
//   * S^T = K Q^T by 32 x 32 MFMA tiles: lane (n, h) gets 16 scores of row n, of the keys 8 (r / 4) + 4 h + r % 4. Largest score and sum of a row are
//     15 steps in the lane and one across lanes n and n + 32.
//   * Those registers are the second product's operand as they stand: O^T = V^T P^T, whose k indices are dealt to the lanes the same way. With 16-bit
//     values V's operand comes from LDS by transposing reads, with float32 by 4-byte reads. Every lane has one row: a running maximum that
//     changes is one factor to a lane.
//   * Keys and values are staged through LDS for all waves, 16-byte pieces permuted within a row so that reads of a column meet no bank twice.
// P is rounded to the arrays' type for the second product, half a step of it; the sum is that of the values before.
// Few rows: the keys are dealt to `splits` workgroups, whose maxima, sums and outputs a second launch joins.
#include "mixed.h"
#include "gemm_tile.h"

#include <algorithm>

namespace mi355x {

typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct DiffArgs {
    const void* Q; const void* K; const void* V; void* O;
    const float* q1; const float* k1; const float* q2; const float* k2;
    const int32_t* lengths;
    float* partial_o; float* partial_ml;   // of splits; [split][slice][row][map][2 d], [split][slice][row][map][2]
    int64_t batch, Sq, Sk;
    int heads, groups, share, vector;   // share = heads / groups; vector: length of the learned vectors
    int causal, splits;
    int64_t row_blocks;                 // of the rows Sq * share of a slice (one batch entry, one group)
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

// A tile's geometry: KT keys of 2 D values (both maps' keys, or the values), in pieces of 16 bytes of which piece c of key k lies at c ^ place(k): a bijection
// of 16 keys (of one piece, as scores read them), and of four keys onto different quarters of the banks (the transposing reads).
template <class T, int D>
struct DiffTile {
    static constexpr int KT = 32, E = 16 / sizeof(T), PIECES = 2 * D / E;   // (8 at least)
    static constexpr int BYTES = KT * 2 * D * (int)sizeof(T);
    static __device__ __forceinline__ int place(int key) { return PIECES == 8 ? (key >> 1 & 1) << 2 | (key >> 2 & 3) : (key & 3) << 2 | (key >> 2 & 3); }
    static __device__ __forceinline__ int at(int key, int piece) { return (key * PIECES + (piece ^ place(key))) * E; }   // in values
};

// One map's operand of Q: D / (2 E) pieces of 16 bytes to a lane.
template <class T, int D>
struct DiffWave {
    using Tile = DiffTile<T, D>;
    static constexpr int E = Tile::E, QP = D / (2 * E), VT = 2 * D / 32;

    typedef T Piece __attribute__((ext_vector_type(E)));
    typedef Piece UnalignedPiece __attribute__((aligned(sizeof(T))));

    // S^T of 32 keys and 32 rows
    static __device__ __forceinline__ f32x16 scores(const T* lds_k, int map, int n, int h, const Piece (&q)[QP]) {
        f32x16 acc = {};
#pragma unroll
        for (int s = 0; s < QP; ++s) {
            const Piece k = *reinterpret_cast<const Piece*>(lds_k + Tile::at(n, map * (D / E) + 2 * s + h));
            if constexpr (std::is_same_v<T, float>) {
#pragma unroll
                for (int e = 0; e < E; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[s][e], acc, 0, 0, 0);
            } else if constexpr (std::is_same_v<T, f16>) {
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[s], acc, 0, 0, 0);
            } else {
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[s], acc, 0, 0, 0);
            }
        }
        return acc;
    }

    // O^T += V^T P^T over 32 keys
    template <int RB>
    static __device__ __forceinline__ void values(const T* lds_v, int n, int h, const f32x16 (&prob)[RB], f32x16 (&out)[RB][VT]) {
        if constexpr (std::is_same_v<T, float>) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = 8 * (r / 4) + 4 * h + r % 4;
#pragma unroll
                for (int c = 0; c < VT; ++c) {
                    const int col = 32 * c + n;
                    const float v = lds_v[Tile::at(key, col / E) + col % E];
#pragma unroll
                    for (int b = 0; b < RB; ++b) out[b][c] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, prob[b][r], out[b][c], 0, 0, 0);
                }
            }
        } else {
            const int lane = threadIdx.x % WAVE, row = lane % 16 / 4, col = 16 * (lane / 16 % 2) + 4 * (lane % 4);   // what a transposing read fetches for others
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Piece pr[RB];
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int e = 0; e < 8; ++e) pr[b][e] = (T)prob[b][8 * t + e];
#pragma unroll
                for (int c = 0; c < VT; ++c) {
                    s16x4 half[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int key = 16 * t + 8 * i + 4 * h + row, value = 32 * c + col;
                        half[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_v + Tile::at(key, value / 8) + value % 8));
                    }
                    const Piece v = __builtin_bit_cast(Piece, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int b = 0; b < RB; ++b) {
                        if constexpr (std::is_same_v<T, f16>) out[b][c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pr[b], out[b][c], 0, 0, 0);
                        else out[b][c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, pr[b], out[b][c], 0, 0, 0);
                    }
                }
            }
        }
    }
};

template <class T, int D, int RB, int RW>
__global__ __launch_bounds__(128 * RW) void diff_attention_kernel(DiffArgs p) {
    using Tile = DiffTile<T, D>;
    using Wave = DiffWave<T, D>;
    using Piece = typename Wave::Piece;
    using UnalignedPiece = typename Wave::UnalignedPiece;
    constexpr int KT = Tile::KT, E = Tile::E, NT = 128 * RW, VT = Wave::VT, ROWS = 32 * RB * RW;
    constexpr int PER_T = KT * Tile::PIECES / NT;
    static_assert(KT * Tile::PIECES % NT == 0, "whole pieces to a thread");
    constexpr int EXCHANGE = 32 * 2 * D * 4;   // bytes of a row block's output
    constexpr int LDS = std::max(2 * Tile::BYTES, RW * EXCHANGE);
    __shared__ __attribute__((aligned(16))) unsigned char lds[LDS];
    T* lds_k = reinterpret_cast<T*>(lds);
    T* lds_v = reinterpret_cast<T*>(lds + Tile::BYTES);

    const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int n = lane % 32, h = lane / 32, map = wave % 2, row_wave = wave / 2;
    const int64_t logical = xcd_remap(blockIdx.x, (int64_t)gridDim.x);
    const int64_t block = logical % p.row_blocks, rest = logical / p.row_blocks;
    const int split = (int)(rest % p.splits);
    const int64_t slice = rest / p.splits, b = slice / p.groups;
    const int group = (int)(slice % p.groups);
    const int64_t rows = p.Sq * p.share, length = diff_length(p, b);
    const int64_t ahead = length - p.Sq;   // if causal, query i sees the keys up to i + ahead

    // ---- queries: row r of a slice is head r % share of query r / share ------------------------------------
    int64_t row[RB], seen[RB];   // seen: keys of the row
    Piece q[RB][Wave::QP];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        row[i] = block * ROWS + (row_wave * RB + i) * 32 + n;
        const int64_t r = row[i] < rows ? row[i] : rows - 1, query = r / p.share;
        const int head = group * p.share + (int)(r % p.share);
        seen[i] = p.causal ? std::max((int64_t)0, std::min(length, query + ahead + 1)) : length;
        const T* from = static_cast<const T*>(p.Q) + ((b * p.Sq + query) * 2 * p.heads + 2 * head + map) * D + h * E;
#pragma unroll
        for (int s = 0; s < Wave::QP; ++s) q[i][s] = *reinterpret_cast<const UnalignedPiece*>(from + 2 * s * E);
    }
    // keys that any row of the workgroup sees, and that the last of its rows sees all of
    const int64_t last = std::min(rows, (block + 1) * ROWS) - 1;
    const int64_t end = p.causal ? std::max((int64_t)0, std::min(length, last / p.share + ahead + 1)) : length;
    const int64_t all = p.causal ? std::max((int64_t)0, std::min(length, block * ROWS / p.share + ahead + 1)) : length;
    const int64_t tiles = (end + KT - 1) / KT, per_split = (tiles + p.splits - 1) / p.splits;
    const int64_t first_tile = split * per_split, end_tile = std::min(tiles, first_tile + per_split);

    const T* K = static_cast<const T*>(p.K) + (b * p.Sk * p.groups + group) * 2 * D;
    const T* V = static_cast<const T*>(p.V) + (b * p.Sk * p.groups + group) * 2 * D;
    const int64_t key_stride = (int64_t)p.groups * 2 * D;

    f32x16 out[RB][VT];
    float most[RB], sum[RB];   // of the scores times scale_log2; the lane's share of the sum
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        most[i] = -__builtin_inff();
        sum[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < VT; ++c) out[i][c] = f32x16{};
    }

    for (int64_t tile = first_tile; tile < end_tile; ++tile) {
        Piece k[PER_T], v[PER_T];
#pragma unroll
        for (int j = 0; j < PER_T; ++j) {
            const int piece = (tid + j * NT) % Tile::PIECES, key = (tid + j * NT) / Tile::PIECES;
            k[j] = v[j] = Piece{};
            if (tile * KT + key < length) {   // (keys that do not exist may lie outside, or hold anything)
                const int64_t at = (tile * KT + key) * key_stride + piece * E;
                k[j] = *reinterpret_cast<const UnalignedPiece*>(K + at);
                v[j] = *reinterpret_cast<const UnalignedPiece*>(V + at);
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER_T; ++j) {
            const int piece = (tid + j * NT) % Tile::PIECES, key = (tid + j * NT) / Tile::PIECES;
            *reinterpret_cast<Piece*>(lds_k + Tile::at(key, piece)) = k[j];
            *reinterpret_cast<Piece*>(lds_v + Tile::at(key, piece)) = v[j];
        }
        __syncthreads();

        f32x16 s[RB];
#pragma unroll
        for (int i = 0; i < RB; ++i) s[i] = Wave::scores(lds_k, map, n, h, q[i]);
        if ((tile + 1) * KT > all) {
#pragma unroll
            for (int i = 0; i < RB; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (tile * KT + 8 * (r / 4) + 4 * h + r % 4 >= seen[i]) s[i][r] = -__builtin_inff();
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            float m = s[i][0];
#pragma unroll
            for (int r = 1; r < 16; ++r) m = fmaxf(m, s[i][r]);
            m = fmaxf(m, __shfl_xor(m, 32, WAVE)) * p.scale_log2;
            if (__any(m > most[i])) {
                const float now = fmaxf(most[i], m), factor = most[i] == now ? 1.0f : __builtin_amdgcn_exp2f(most[i] - now);
                most[i] = now;
                sum[i] *= factor;
#pragma unroll
                for (int c = 0; c < VT; ++c) out[i][c] *= factor;
            }
            const float base = most[i] == -__builtin_inff() ? 0.0f : most[i];   // no key so far: exp2(-inf)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[i][r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], p.scale_log2, -base));
                sum[i] += s[i][r];
            }
        }
        Wave::values(lds_v, n, h, s, out);
    }

    // ---- the two maps meet --------------------------------------------------------------------------------
    float* exchange = reinterpret_cast<float*>(lds) + row_wave * (EXCHANGE / 4);
    const float weight = p.splits > 1 ? 0.0f : diff_lambda(p);
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        sum[i] += __shfl_xor(sum[i], 32, WAVE);
        if (p.splits > 1) {
            if (row[i] < rows) {
                const int64_t at = ((split * p.batch * p.groups + slice) * rows + row[i]) * 2 + map;
                if (h == 0) {
                    p.partial_ml[2 * at] = most[i];
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
        __syncthreads();
        if (map == 1) {
#pragma unroll
            for (int c = 0; c < VT; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) exchange[(16 * c + r) * WAVE + lane] = out[i][c][r] * factor;
        }
        __syncthreads();
        if (map == 0 && row[i] < rows) {
            const int64_t query = row[i] / p.share;
            const int head = group * p.share + (int)(row[i] % p.share);
            T* to = static_cast<T*>(p.O) + ((b * p.Sq + query) * p.heads + head) * 2 * D;
#pragma unroll
            for (int c = 0; c < VT; ++c)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = out[i][c][4 * g + e] * factor - exchange[(16 * c + 4 * g + e) * WAVE + lane];
                    store_values(to + 32 * c + 8 * g + 4 * h, o, 4);
                }
        }
    }
}

// The splits of a row joined: one wave to a row, its lanes the 2 D values.
template <class T, int D>
__global__ __launch_bounds__(256) void diff_join_kernel(DiffArgs p) {
    constexpr int PER_LANE = 2 * D / WAVE;
    const int64_t rows = p.Sq * p.share, all = p.batch * p.groups * rows;
    const int64_t at = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;   // of a slice's row
    const int lane = threadIdx.x % WAVE;
    if (at >= all) return;
    const float weight = diff_lambda(p);
    float result[PER_LANE] = {};
#pragma unroll
    for (int map = 0; map < 2; ++map) {
        float most = -__builtin_inff();
        for (int s = 0; s < p.splits; ++s) most = fmaxf(most, p.partial_ml[2 * ((s * all + at) * 2 + map)]);
        const float base = most == -__builtin_inff() ? 0.0f : most;
        float sum = 0.0f, o[PER_LANE] = {};
        for (int s = 0; s < p.splits; ++s) {
            const int64_t i = (s * all + at) * 2 + map;
            const float factor = __builtin_amdgcn_exp2f(p.partial_ml[2 * i] - base);
            sum = fmaf(p.partial_ml[2 * i + 1], factor, sum);
#pragma unroll
            for (int e = 0; e < PER_LANE; ++e) o[e] = fmaf(p.partial_o[i * 2 * D + lane * PER_LANE + e], factor, o[e]);
        }
        const float factor = sum == 0.0f ? 0.0f : (map ? -weight : 1.0f) / sum;
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) result[e] += o[e] * factor;
    }
    const int64_t slice = at / rows, row = at % rows, b = slice / p.groups;
    const int head = (int)(slice % p.groups) * p.share + (int)(row % p.share);
    store_values(static_cast<T*>(p.O) + ((b * p.Sq + row / p.share) * p.heads + head) * 2 * D + lane * PER_LANE, result, PER_LANE);
}

template <class T, int D>
static int launch_diff(DiffArgs p, hipStream_t st) {
    constexpr int RB = D * sizeof(T) <= 128 ? 2 : 1, RW = 2;
    const int64_t rows = p.Sq * p.share;
    p.row_blocks = ceil_div(rows, (int64_t)(32 * RB * RW));
    const int64_t grid = p.row_blocks * p.splits * p.batch * p.groups;
    MI355X_REQUIRE(grid_fits(grid, 128 * RW), "differential_attention: too large");
    hipLaunchKernelGGL((diff_attention_kernel<T, D, RB, RW>), dim3((unsigned)grid), dim3(128 * RW), 0, st, p);
    if (p.splits > 1) {
        const int64_t all = p.batch * p.groups * rows;
        hipLaunchKernelGGL((diff_join_kernel<T, D>), dim3((unsigned)ceil_div(all, (int64_t)4)), dim3(256), 0, st, p);
    }
    return check_launch("diff_attention_kernel");
}

}  // namespace mi355x

extern "C" int64_t mi355x_differential_attention_splits(int64_t batch, int64_t Sq, int64_t Sk, int64_t heads, int64_t groups, int64_t size, int type) {
    (void)batch; (void)Sq; (void)Sk; (void)heads; (void)groups; (void)size; (void)type;
    return 1;
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
    MI355X_REQUIRE(Sq < (int64_t)1 << 31 && Sk < (int64_t)1 << 31 && heads < 1 << 20 && vector < 1 << 20 && batch < (int64_t)1 << 31, "differential_attention: too large");
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
