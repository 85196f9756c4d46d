// A wave's part of attention by 32 x 32 tiles of the matrix unit: keys and values in LDS, scores, and the product of the probabilities with the values.
#pragma once

#include "mixed.h"
#include "gemm_tile.h"

namespace mi355x {

typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// f(a lane's value, that of the lane 32 from it)
template <class F>
__device__ __forceinline__ float across_halves(float v, F&& f) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const auto both = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);   // the lower lanes' values, the upper lanes'
    const uint32_t lower = both[0], upper = both[1];   // (a bit_cast of a vector's element is one of its first)
    return f(__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper));
}

// Where keys and values, rows of W values each, lie in LDS: rows of 16-byte pieces, of which piece c of key k lies at c ^ place(k): a bijection
// of 16 keys (of one piece, as scores read them), and of four keys onto different quarters of the banks (the transposing reads).
template <class T, int W>
struct AttentionTile {
    static constexpr int E = 16 / sizeof(T), PIECES = W / E, ROW = W * (int)sizeof(T);   // (8 pieces at least)
    static __device__ __forceinline__ int place(int key) { return PIECES == 8 ? (key >> 1 & 1) << 2 | (key >> 2 & 3) : (key & 3) << 2 | (key >> 2 & 3); }
    static __device__ __forceinline__ int at(int key, int piece) { return (key * PIECES + (piece ^ place(key))) * E; }   // in values
};

// 16 bytes to a lane from global memory, base + the lane's offset, into LDS at lds + 16 lane; base and lds are the same for the wave.
__device__ __forceinline__ void attention_to_lds(const void* base, uint32_t offset, uint32_t lds) {
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const uint64_t uniform = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(offset), "s"(uniform) : "memory", "m0");
}

// Eight values of an operand as the matrix unit takes them: one vector of 16-bit numbers, or a float32 as the sum of three bfloat16 numbers, its
// first, middle and last eight bits, cut off one after the other: all of its sign. Of the nine partial products of two such values the six largest are taken; those left out are
// below 2^-21 of the product (both values 1 + 2^-7 - 2^-23: 2^-21.0; 2^-24.5 on average), always towards zero. Parts to the nearest would leave half of that and less to either
// side, but the first part of values from 2^128 - 2^119 on would be infinite. (An infinity is no such sum: it gives NaN.)
template <class T>
struct Operand {
    typedef T Vector __attribute__((ext_vector_type(8)));
    Vector part[1];
    __device__ __forceinline__ void set(const T (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) part[0][e] = v[e];
    }
    // sum + the eight values as they are rounded, two to an instruction
    __device__ __forceinline__ void add_to(float& sum, const T (&)[8]) const {
        typedef T Pair __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const Pair two = {part[0][e], part[0][e + 1]};
            if constexpr (std::is_same_v<T, f16>) sum = __builtin_amdgcn_fdot2(two, Pair{(T)1.0f, (T)1.0f}, sum, false);
            else sum = __builtin_amdgcn_fdot2_f32_bf16(two, Pair{(T)1.0f, (T)1.0f}, sum, false);
        }
    }
    static __device__ __forceinline__ void product(const Operand& a, const Operand& b, f32x16& acc) {
        if constexpr (std::is_same_v<T, f16>) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.part[0], b.part[0], acc, 0, 0, 0);
        else acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.part[0], b.part[0], acc, 0, 0, 0);
    }
};
template <>
struct Operand<float> {
    u32x4 part[3];
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x[2] = {v[2 * e], v[2 * e + 1]};
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const uint32_t bits[2] = {__builtin_bit_cast(uint32_t, x[0]), __builtin_bit_cast(uint32_t, x[1])};
                part[i][e] = __builtin_amdgcn_perm(bits[1], bits[0], 0x07060302u);   // the upper halves
                if (i == 2) break;
#pragma unroll
                for (int j = 0; j < 2; ++j) x[j] -= __builtin_bit_cast(float, bits[j] & 0xffff0000u);
            }
        }
    }
    __device__ __forceinline__ void add_to(float& sum, const float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += v[e];
    }
    static __device__ __forceinline__ void product(const Operand& a, const Operand& b, f32x16& acc) {
        auto one = [&](int i, int j) __attribute__((always_inline)) {
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.part[i]), __builtin_bit_cast(bf16x8, b.part[j]), acc, 0, 0, 0);
        };
        one(0, 2), one(1, 1), one(2, 0), one(0, 1), one(1, 0), one(0, 0);   // the smallest first
    }
};

// Queries and keys of D values, of which a row of W holds W / D (maps); values of W, of which the wave has COLUMNS
template <class T, int W, int D, int COLUMNS = W>
struct AttentionWave {
    using Tile = AttentionTile<T, W>;
    static constexpr int E = Tile::E, QP = D / 16, VT = COLUMNS / 32;   // operands of a map's query or key, tiles of 32 value columns

    typedef T Piece __attribute__((ext_vector_type(E)));
    typedef Piece UnalignedPiece __attribute__((aligned(sizeof(T))));

    // Addresses in LDS of what a lane reads differ by constants in the bits of the piece (an exclusive or) and in those of the key (an offset of the
    // instruction). Two of them are kept and the others made where they are used: kept as well they took 64 registers, and the accumulators went to memory.
    template <class V>
    static __device__ __forceinline__ V read(uint32_t at, int offset) {
        return *reinterpret_cast<const __attribute__((address_space(3))) V*>(reinterpret_cast<const __attribute__((address_space(3))) char*>(at) + offset);
    }
    static __device__ __forceinline__ uint32_t key_address(int map, int n, int h) { return Tile::at(n, (map * D + 8 * h) / E) * sizeof(T); }
    static __device__ __forceinline__ uint32_t value_address(int lane, int n, int h) {
        if constexpr (std::is_same_v<T, float>) return Tile::at(4 * h, n / E) * sizeof(T) + n % E * sizeof(T);
        const int row = lane % 16 / 4, col = 16 * (lane / 16 % 2) + 4 * (lane % 4);   // what a transposing read fetches for others
        return Tile::at(4 * h + row, col / 8) * sizeof(T) + col % 8 * sizeof(T);
    }

    // use(i, operand) for operands i = 0 .. N - 1, MFMAS products each. Of float32, which takes 44 instructions to split, operand i + 1 is split between the products of
    // operand i, and operand i + 2 is on its way from LDS: a wave issues in order, and a product holds the matrix unit for the time of seven instructions.
    template <int N, int MFMAS, class Read, class Use>
    static __device__ __forceinline__ void each_operand(Read&& fetch, Use&& use) {
        if constexpr (!std::is_same_v<T, float>) {
            static_for<N>([&](auto i) __attribute__((always_inline)) {
                Operand<T> v;
                fetch(i, v.part[0]);
                use(i, v);
            });
        } else {
            float x[8];
            Operand<T> now;
            fetch(Int<0>{}, x);
            now.set(x);
            if constexpr (N > 1) fetch(Int<1>{}, x);
            static_for<N>([&](auto i) __attribute__((always_inline)) {
                constexpr int I = decltype(i)::value;
                float y[8];
                Operand<T> next;
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (I + 2 < N) fetch(Int<I + 2>{}, y);
                if constexpr (I + 1 < N) next.set(x);
                use(i, now);
                __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);   // LDS reads
                static_for<MFMAS>([&](auto) __attribute__((always_inline)) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                  // a product
                    __builtin_amdgcn_sched_group_barrier(0x002, 48 / MFMAS + 1, 0);   // other arithmetic
                });
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (I + 1 < N) now = next;
                if constexpr (I + 2 < N) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = y[e];
                }
            });
        }
    }

    // S^T of 32 keys and 32 rows
    template <int RB>
    static __device__ __forceinline__ void scores(uint32_t lds_k, const Operand<T> (&q)[RB][QP], f32x16 (&acc)[RB]) {
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = f32x16{};
        each_operand<QP, 6 * RB>(
            [&](auto s, auto& v) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 8 / E; ++i) {
                    const Piece piece = read<Piece>(lds_k ^ (16 * (16 / E * decltype(s)::value + i)), 0);
#pragma unroll
                    for (int e = 0; e < E; ++e) v[i * E + e] = piece[e];
                }
            },
            [&](auto s, const Operand<T>& k) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < RB; ++b) Operand<T>::product(k, q[b][decltype(s)::value], acc[b]);
            });
    }

    // O^T += V^T P^T and the lane's share of the rows' sums of P over 32 keys; element e of half h of a k-step t is key 16 t + 4 h + e, from e = 4 on four more
    template <int RB>
    static __device__ __forceinline__ void values(uint32_t lds_v, const f32x16 (&prob)[RB], f32x16 (&out)[RB][VT], float (&sum)[RB]) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            Operand<T> pr[RB];
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                T v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = (T)prob[b][8 * t + e];
                pr[b].set(v);
                pr[b].add_to(sum[b], v);
            }
            each_operand<VT, 6 * RB>(
                [&](auto column, auto& v) __attribute__((always_inline)) {
                    constexpr int c = decltype(column)::value;
                    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = read<float>(lds_v ^ (16 * (8 * c ^ (e % 4) << 2 ^ 2 * (e / 4))), (16 * t + 8 * (e / 4) + e % 4) * Tile::ROW);
                    } else {
                        s16x4 half[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            half[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(reinterpret_cast<__attribute__((address_space(3))) char*>(
                                lds_v ^ (16 * (4 * c ^ 2 * i))) + (16 * t + 8 * i) * Tile::ROW));
                        v = __builtin_bit_cast(typename Operand<T>::Vector, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
                    }
                },
                [&](auto column, const Operand<T>& v) __attribute__((always_inline)) {
#pragma unroll
                    for (int b = 0; b < RB; ++b) Operand<T>::product(v, pr[b], out[b][decltype(column)::value]);
                });
        }
    }
};

}  // namespace mi355x
