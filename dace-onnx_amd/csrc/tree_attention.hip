// TreeAttention: O = softmax(c Q K^T) V over a cache in pages, whose last tokens are a chain or a tree. The reference has no such node.
//
// Rows: a slice (an entry's group of keys and values) has tokens * share of them, the heads that share it side by side, so a page is read once for all of them. A workgroup has 64 or 128
// rows and walks the keys in stages of 32, 64 or 128, from the end on: S^T = K Q^T and O^T = V^T P^T by products of 32 x 32 x 16, in which a lane has a row of its own, its maximum and sum
// included; P goes from one product to the next in registers. Softmax runs in powers of two: a row has a base b, P = 2^(c' s - b) with c' = c log2 e, and sums and outputs take a factor where
// the base moves. Scores, bases, sums and outputs are float32; with arrays of 16 bits P is rounded to their type for its product, by half a step of it, and its sum is taken of the rounded
// values, so that weights add up to 1. float32 goes by three bfloat16 parts of each operand and the six largest products of them; those left out are below 2^-21 of the product.
// Whom a row sees: of the keys in front of the call all, of the call's its ancestors. Those fall, so a row walking back through the keys holds the next one and looks each up once in
// a table of parents in LDS: a mask of 32 bits for 32 keys, taken where a block holds keys that some row does not see, nowhere else. Values that are not finite become 0 there, as 0 times
// one is not a number, and the rows that do see them add them one by one.
// Keys and values come from their pages into a ring of stages in LDS by transfers of 1 KB that no register waits for; a wave's transfer knows its page by a scalar load, and where pages are long
// enough two to eight transfers share one. (Pages that are no whole number of transfers: through registers.)
// Few rows and long caches leave CUs without work: the keys of all blocks are then cut into parts that are dealt to a fixed number of workgroups, by the lengths that the kernel finds, not by
// the table's room, and a second kernel joins the parts' outputs by their bases and sums. What the first says about the cut stands in scratch memory. There are as many
// workgroups as are resident, and keys are cut where no more blocks than that (and 256 entries) are: beyond, a block is one workgroup's, however long. That is behind where one entry is far longer than the
// others: one token for each of 64 entries, 63 behind 1000 and one behind 131072, 32 heads in 8 groups of 128: 2150 us, where bytes take 156 (16 of them 114 and 117; 64 behind 1000 53 and 52).
// No atomics but those that mark keys: results repeat.
//
// Bound, at heads of 128 in bfloat16 (a copy 5.1 TB/s, a product of 8192^3 1570 TFLOP/s):
// - one token, 16 entries of up to 8192, 32 heads in 8 groups: bytes. 69 to 71 us, 5.2 TB/s; one token of 16 heads in 4 groups behind 131072, in float16, 55 us, 4.9 TB/s, the join 5 of them.
// - a prompt of 4096 behind 4096, 16 heads in 4 groups: products and powers, 214 to 231 us, 890 to 960 TFLOP/s. Of a wave's cycles 42 % issue, 34 % wait for a unit, 25 % for LDS and barriers;
//   the matrix unit is busy for 48 % of the time in which its CU has work, which is 87 %: the longest block ends last, the second half of it with its CU to itself. The vector instructions of 32
//   keys (a power, a multiply-add, half a conversion and half a product of pairs for each score) take about as long as their products, and the products of a wave's own are where they hide
//   best (below). With 256 rows to a workgroup, one to a CU, calls whose blocks are all as long take 5 % less, but causal ones 11 % more: no short block stands next to a long one.
// - 4 trees of 32 behind up to 4096, 32 heads in 8 groups: 26 us where bytes are 9, 21 of them in the first kernel and 5.4 in the second. A workgroup has about six stages, and what each waits for comes
//   one after the other: its part, its pages, the first keys, the parts' sums. 128 rows read every key once.
#include "attention_tile.h"

#include <algorithm>

namespace mi355x {

constexpr int TREE_MOST = 1024;   // tokens of a tree
constexpr float LOG2_E = 1.44269504088896340736f;

struct TreeArgs {
    const void* q; const void* k_pages; const void* v_pages; const int32_t* table; const int32_t* lengths; const int32_t* parents; void* o;
    float* partial_o; float* partial_ml;   // of parts: [workgroup][row of the block][D], [workgroup][row of the block][2]
    int32_t* plan;                         // [entry][2]: its first workgroup, the parts of its blocks
    int64_t batch, tokens, columns, row_blocks;
    int pages, page_size, capacity;        // capacity = page_size * columns
    int heads, kv_heads, share;            // share = heads / kv_heads
    int block_rows;                        // of a workgroup's part
    int dealt;                             // workgroups that the parts of all blocks are dealt to; 0: one workgroup to a block
    int order;                             // with one workgroup to a block: see tree_block
    uint32_t page_magic; int page_shift;   // n / page_size for n below 2^31
    float scale_log2;
};

__device__ __forceinline__ int tree_column(const TreeArgs& p, int n) { return (int)(__umulhi(2u * (uint32_t)n, p.page_magic) >> p.page_shift); }

struct TreeEntry { int length, total; };   // keys before the call, and with it
__device__ __forceinline__ TreeEntry tree_entry(const TreeArgs& p, int64_t b) {
    const int given = p.lengths[b], length = given < 0 ? 0 : given > p.capacity ? p.capacity : given;
    return {length, (int)std::min<int64_t>(length + p.tokens, p.capacity)};
}

// What a row whose weights add up to 0 is scaled by: one without keys is 0, one whose scores are all minus infinity is not a number. Without keys in front of the call a row has one if the token
// that its line begins with has a column; a line falls, whatever parent(token) says.
template <class Parent>
__device__ __forceinline__ float tree_no_weights(const TreeArgs& p, const TreeEntry& entry, int token, Parent&& parent) {
    int first = 0;
    if (p.parents && entry.length == 0 && entry.total > 0) {
        first = token;
        for (int up = parent(first); up >= 0 && up < first; up = parent(first)) first = up;
    }
    return entry.length > 0 || first < entry.total ? __builtin_nanf("") : 0.0f;
}

// f over the lanes of a wave, four of a row at a time, then the rows; every lane gets it
template <class F>
__device__ __forceinline__ uint32_t wave_uint(uint32_t v, F&& f) {
    auto across = [&](auto control) { v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(control)::value, 0xf, 0xf, false)); };
    across(Int<DPP_QUAD_XOR1>{}), across(Int<DPP_QUAD_XOR2>{}), across(Int<DPP_ROW_HALF_MIRROR>{}), across(Int<DPP_ROW_MIRROR>{});
    auto row = [&](int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); };
    return f(f(row(0), row(16)), f(row(32), row(48)));
}

// v of a lane and those before it: by rows of sixteen lanes, then the rows' ends to the rows behind them
__device__ __forceinline__ int wave_sums(int v) {
    auto from = [&](auto control, auto rows) { v += __builtin_amdgcn_update_dpp(0, v, decltype(control)::value, decltype(rows)::value, 0xf, false); };
    from(Int<0x111>{}, Int<0xf>{}), from(Int<0x112>{}, Int<0xf>{}), from(Int<0x114>{}, Int<0xf>{}), from(Int<0x118>{}, Int<0xf>{});   // row_shr:1, 2, 4, 8
    from(Int<0x142>{}, Int<0xa>{}), from(Int<0x143>{}, Int<0xc>{});                                                                   // row_bcast:15, 31
    return v;
}

// The keys of every block of an entry, in stages of KT, cut into as many parts as it takes for none to have more than `most` stages, which is as few as leave enough workgroups for all
// parts; an entry's `items` blocks count alike. Workgroups go by entry, block and part. A lane of each wave looks at entries lane, lane + 64, ...
constexpr int DEAL_ENTRIES = 256;
template <int KT>
struct TreeDeal {
    static constexpr int EACH = DEAL_ENTRIES / WAVE;
    int64_t items;   // blocks of an entry
    uint32_t most, stages[EACH];
    __device__ __forceinline__ uint32_t parts(uint32_t stages) const { return (stages + most - 1) / most; }
    __device__ __forceinline__ int64_t all_parts(const TreeArgs& p) const {
        int64_t all = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (i * WAVE >= p.batch) break;
            all += wave_uint(parts(stages[i]), [](uint32_t x, uint32_t y) { return x + y; });
        }
        return all;
    }
    __device__ __forceinline__ TreeDeal(const TreeArgs& p) : items(p.kv_heads * p.row_blocks) {
        int64_t all = 0;
        uint32_t longest = 1;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int64_t b = i * WAVE + threadIdx.x % WAVE;
            stages[i] = b < p.batch ? std::max(1, (tree_entry(p, b).total + KT - 1) / KT) : 0;
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (i * WAVE >= p.batch) break;
            all += wave_uint(stages[i], [](uint32_t x, uint32_t y) { return x + y; });
            longest = std::max(longest, wave_uint(stages[i], [](uint32_t x, uint32_t y) { return x > y ? x : y; }));
        }
        // Between what even parts without a remainder would take and where a part more for every block cannot be too many, both a little wide as they are taken in float32; the longest is
        // always enough: there are no more blocks than workgroups.
        const float work = (float)all * (float)items, spare = (float)(p.dealt - (int)(p.batch * items));
        uint32_t low = std::max(1u, (uint32_t)(work / (float)p.dealt * (1.0f - 0x1p-20f)));
        most = spare > 0.0f ? std::min(longest, (uint32_t)std::min(0x1p31f, work / spare * (1.0f + 0x1p-20f) + 1.0f)) : longest;
        while (low < most) {
            const uint32_t enough = most;
            most = low + (enough - low) / 2;
            if (all_parts(p) * items <= p.dealt) continue;
            low = most + 1;
            most = enough;
        }
    }
    // the entry that workgroup w is of, which of the entry's it is, and how many parts the entry's blocks have; false: of none
    __device__ __forceinline__ bool find(const TreeArgs& p, int64_t w, int64_t& b, int64_t& of_entry, int& own) const {
        int64_t passed = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (i * WAVE >= p.batch) break;
            const int mine = (int)parts(stages[i]);
            const int with = wave_sums(mine);
            const uint64_t beyond = __ballot((passed + with) * items > w);
            if (beyond) {
                const int lane = __builtin_ctzll(beyond);
                own = __builtin_amdgcn_readlane(mine, lane);
                b = i * WAVE + lane;
                of_entry = w - (passed + __builtin_amdgcn_readlane(with, lane) - own) * items;
                return true;
            }
            passed += __builtin_amdgcn_readlane(with, WAVE - 1);
        }
        return false;
    }
};

// Which block of a call that is not dealt out workgroup blockIdx.x has. The hardware deals workgroups to the XCDs in turn, and those of an XCD to its CUs in turn: slices (an
// entry's group) stay on one XCD or few, whose L2 their keys then pass once, and every XCD has blocks of all lengths.
// order 0: the long ones first; 1: of up to two workgroups to a CU, a long one and a short one.
__device__ __forceinline__ void tree_block(const TreeArgs& p, int64_t& slice, int64_t& block) {
    const int64_t slices = p.batch * p.kv_heads, grid = slices * p.row_blocks;
    const uint32_t w = blockIdx.x;
    int64_t turn;
    if (slices % NUM_XCD == 0) {
        const uint32_t each = (uint32_t)(slices / NUM_XCD), local = w / NUM_XCD;
        slice = w % NUM_XCD * (int64_t)each + local % each;
        turn = local / each;
    } else {
        slice = w % slices;
        turn = w / slices;
    }
    if (p.order && turn * slices >= grid / 2) turn = p.row_blocks - 1 - (turn - (grid / 2 + slices - 1) / slices);
    block = p.row_blocks - 1 - turn;
}

// the lowest n of 32 bits
__device__ __forceinline__ uint32_t lowest_bits(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }

// N KB of keys or values that lie one behind the other, to LDS likewise: the offset of an instruction counts on both sides
template <int N>
__device__ __forceinline__ void run_to_lds(const void* base, const uint32_t* lane_offset, uint32_t lds) {
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const uint64_t uniform = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
    const int to = __builtin_amdgcn_readfirstlane((int)lds);
    static_assert(N == 1 || N == 2 || N == 4, "offsets of 12 bits");
    if constexpr (N == 1)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(lane_offset[0]), "s"(uniform) : "memory", "m0");
    else if constexpr (N == 2)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024" ::"s"(to), "v"(lane_offset[0]),
                     "v"(lane_offset[1]), "s"(uniform) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\tglobal_load_lds_dwordx4 %2, %5 offset:1024\n\tglobal_load_lds_dwordx4 %3, %5 offset:2048\n\t"
                     "global_load_lds_dwordx4 %4, %5 offset:%6" ::"s"(to), "v"(lane_offset[0]), "v"(lane_offset[1]), "v"(lane_offset[2]), "v"(lane_offset[3]), "s"(uniform), "n"(3 * 1024) : "memory", "m0");
}

template <class T, int D, int BATCH>
__device__ __forceinline__ void tree_read_keys(uint32_t lds_k, int s0, typename Values<T, 8>::vec (&k)[BATCH]) {
#pragma unroll
    for (int s = 0; s < BATCH; ++s) k[s] = AttentionWave<T, D, D>::template read<typename Values<T, 8>::vec>(lds_k ^ (32 * (s0 + s)), 0);
}

// S^T of 32 keys and 32 rows; between(s): what else goes on behind product s
template <class T, int D, int BATCH, class F>
__device__ __forceinline__ void tree_scores(uint32_t lds_k, typename Values<T, 8>::vec (&k)[BATCH], const Operand<T> (&q)[D / 16], f32x16& acc, F&& between) {
    acc = f32x16{};
#pragma unroll
    for (int s0 = 0; s0 < D / 16; s0 += BATCH) {
        if (s0) tree_read_keys<T, D, BATCH>(lds_k, s0, k);
#pragma unroll
        for (int s = 0; s < BATCH; ++s) {
            Operand<T>::product({{k[s]}}, q[s0 + s], acc);
            between(s0 + s);
        }
    }
}

// (the wave's for blocks of rows, of which it has one)
template <int D>
__device__ __forceinline__ void tree_scores_f32(uint32_t lds_k, const Operand<float> (&q)[D / 16], f32x16& acc) {
    AttentionWave<float, D, D>::scores(lds_k, reinterpret_cast<const Operand<float>(&)[1][D / 16]>(q), reinterpret_cast<f32x16(&)[1]>(acc));
}

// The values' operands of 32 keys: in registers by the time the probabilities are
template <class T, int D, int VT>
__device__ __forceinline__ void tree_read_values(uint32_t lds_v, typename Values<T, 8>::vec (&v)[2 * VT]) {
    constexpr int ROW = AttentionTile<T, D>::ROW;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int c = 0; c < VT; ++c) {
            s16x4 half[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                half[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(reinterpret_cast<__attribute__((address_space(3))) char*>(
                    lds_v ^ (16 * (4 * c ^ 2 * i))) + (16 * t + 8 * i) * ROW));
            v[t * VT + c] = __builtin_bit_cast(typename Values<T, 8>::vec, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
}

// between(n): behind product n of 2 VT
template <class T, int VT, class F>
__device__ __forceinline__ void tree_values(const typename Values<T, 8>::vec (&v)[2 * VT], const f32x16& prob, f32x16 (&out)[VT], float& sum, F&& between) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        Operand<T> pr;
        T x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (T)prob[8 * t + e];
        pr.set(x);
#pragma unroll
        for (int c = 0; c < VT; ++c) {
            Operand<T>::product({{v[t * VT + c]}}, pr, out[c]);
            if (c == 0) {
                pr.add_to(sum, x);
                asm volatile("" : "+v"(sum));   // (taken here, not behind all products)
            }
            between(t * VT + c);
        }
    }
}

// Of float32: the products of 32 keys have sums of their own, which are added to the outputs. The matrix unit loses a little of every sum it adds to, towards zero: outputs of 10000 keys were
// off by 4.7e-6 (2-norm) where all products went to one sum, of 60000 by 1.3e-5; so 2.4e-7 and 3.3e-7, for 1 to 5 % of the time. The sum of the probabilities keeps what its additions lose.
template <int D, int VT>
__device__ __forceinline__ void tree_values_f32(uint32_t lds_v, const f32x16& prob, f32x16 (&out)[VT], float& sum, float& lost) {
    constexpr int ROW = AttentionTile<float, D>::ROW;
    Operand<float> pr[2];
    float all = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = prob[8 * t + e];
        pr[t].set(x);
        pr[t].add_to(all, x);
    }
    const float before = sum, added = before + all - before;
    sum = before + all;
    lost += (before - (sum - added)) + (all - added);
    f32x16 acc[2];
    AttentionWave<float, D, D>::template each_operand<2 * VT, 6>(
        [&](auto operand, auto& v) __attribute__((always_inline)) {
            constexpr int c = decltype(operand)::value / 2, t = decltype(operand)::value % 2;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = AttentionWave<float, D, D>::template read<float>(lds_v ^ (16 * (8 * c ^ (e % 4) << 2 ^ 2 * (e / 4))), (16 * t + 8 * (e / 4) + e % 4) * ROW);
        },
        [&](auto operand, const Operand<float>& v) __attribute__((always_inline)) {
            constexpr int c = decltype(operand)::value / 2, t = decltype(operand)::value % 2;
            if constexpr (t == 0) acc[c % 2] = f32x16{};
            Operand<float>::product(v, pr[t], acc[c % 2]);
            if constexpr (t == 0 && c > 0) out[c - 1] += acc[(c + 1) % 2];   // (those of the columns before: nobody waits for these)
            if constexpr (t == 1 && c == VT - 1) out[c] += acc[c % 2];
        });
}

// Waves: RW blocks of 32 rows, CW shares of the value columns (each takes the scores for itself), KW shares of a stage's keys, 32 SUB each; NS stages. WHOLE: no transfer's keys lie in
// two pages.
template <class T, int D, int RW, int CW, int KW, int SUB, int NS, int PER_SIMD, bool WHOLE>
__global__ __launch_bounds__(64 * RW * CW * KW, PER_SIMD) void tree_attention_kernel(TreeArgs p) {
    using Tile = AttentionTile<T, D>;
    using Wave = AttentionWave<T, D, D, D / CW>;
    using Piece = typename Wave::Piece;
    using UnalignedPiece = typename Wave::UnalignedPiece;
    constexpr int KT = 32 * KW * SUB, E = Tile::E, NT = 64 * RW * CW * KW, VT = Wave::VT, ROWS = 32 * RW;
    constexpr int HALF = KT * Tile::ROW, STAGE = 2 * HALF;            // keys, then values
    constexpr int PER_T = KT * Tile::PIECES / NT, KPT = WAVE / Tile::PIECES;   // transfers of a wave's keys in a stage, keys to a transfer
    static_assert(KT * Tile::PIECES % NT == 0 && Tile::PIECES <= WAVE && NS >= 2 && (NS - 2) * 2 * PER_T < 64, "whole pieces to a thread, whole keys to a transfer");
    constexpr int EXCHANGE = 32 * D / CW;   // floats of a wave's output
    constexpr bool AHEAD = sizeof(T) == 2;   // operands are read from LDS all at once, before they are needed
    __shared__ __attribute__((aligned(1024))) unsigned char lds[std::max(NS * STAGE, KW == 1 ? 0 : 4 * EXCHANGE * (KW / 2) * RW * CW)];
    __shared__ int16_t parents[TREE_MOST];
    __shared__ uint32_t odd_keys[2][KT / 32];   // of the stage and the one before

    const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int n = lane % 32, h = lane / 32, row_wave = wave % RW, column_wave = wave / RW % CW, key_wave = wave / (RW * CW);
    const int64_t rows = p.tokens * p.share;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds;
    const uint32_t key_at = Wave::key_address(0, n, h), value_at = Wave::value_address(lane, n, h) ^ (uint32_t)(column_wave * VT * 32 * sizeof(T));
    if (tid < KT / 32) odd_keys[0][tid] = odd_keys[1][tid] = 0;

    // Piece `lane` of transfer j of a wave, whose keys are one behind the other: where it is, counted from the transfer's first key
    uint32_t offset[PER_T];
#pragma unroll
    for (int j = 0; j < PER_T; ++j) {
        const int key = (wave * PER_T + j) * KPT + lane / Tile::PIECES;
        offset[j] = (uint32_t)(lane / Tile::PIECES * Tile::ROW + (lane % Tile::PIECES ^ Tile::place(key)) * 16);
    }

    int64_t b, block, of_entry;
    int group, part = 0, parts = 1;
    if (p.dealt) {
        const TreeDeal<KT> deal(p);
        if (!deal.find(p, blockIdx.x, b, of_entry, parts)) return;
        if (of_entry == 0 && tid == 0) p.plan[2 * b] = (int32_t)blockIdx.x, p.plan[2 * b + 1] = parts;
        part = (int)(of_entry % parts);
        group = (int)(of_entry / parts / p.row_blocks);
        block = of_entry / parts % p.row_blocks;
    } else {
        int64_t slice;
        tree_block(p, slice, block);
        b = slice / p.kv_heads;
        group = (int)(slice % p.kv_heads);
    }
    const TreeEntry entry = tree_entry(p, b);
    const int length = __builtin_amdgcn_readfirstlane(entry.length), total = __builtin_amdgcn_readfirstlane(entry.total);
    // keys up to and with token `row / share`
    auto up_to = [&](int64_t row) { return (int)std::min<int64_t>(total, length + row / p.share + 1); };
    if (p.parents) {
        for (int i = tid; i < (int)p.tokens; i += NT) {
            const int parent = p.parents[b * p.tokens + i];
            parents[i] = (int16_t)(parent >= 0 && parent < i ? parent : -1);
        }
    }
    // keys that any row of the workgroup sees, and that all of them see; the same of the wave
    const int64_t row0 = block * ROWS + row_wave * 32;   // of the wave
    const int end = up_to(std::min(rows, (block + 1) * ROWS) - 1), all = p.parents ? length : up_to(block * ROWS);
    const int wave_end = row0 < rows ? __builtin_amdgcn_readfirstlane(up_to(std::min(rows, row0 + 32) - 1)) : 0;
    const int wave_all = p.parents ? length : __builtin_amdgcn_readfirstlane(up_to(std::min(rows - 1, row0)));
    const int stages = (end + KT - 1) / KT, first = (int)((int64_t)part * stages / parts), last = (int)((int64_t)(part + 1) * stages / parts), count = last - first;

    // ---- keys and values -------------------------------------------------------------------------------
    typedef const __attribute__((address_space(4))) int32_t Uniform;   // (read by scalar loads, which the transfers' counter does not count)
    const int32_t* const columns = p.table + b * p.columns;
    Uniform* const table = (Uniform*)(uintptr_t)columns;
    const int64_t page_bytes = (int64_t)p.kv_heads * p.page_size * Tile::ROW;
    const char* K = static_cast<const char*>(p.k_pages) + (int64_t)group * p.page_size * Tile::ROW;
    const char* V = static_cast<const char*>(p.v_pages) + (int64_t)group * p.page_size * Tile::ROW;
    auto from_page = [&](int page, int row) { return std::min(std::max(page, 0), p.pages - 1) * page_bytes + (int64_t)row * Tile::ROW; };
    int next_page[PER_T];
    // f(transfers of a wave that are sure to lie in one page, one behind the other)
    auto by_runs = [&](auto&& f) __attribute__((always_inline)) {
        if constexpr (PER_T >= 8) { if (p.page_size % (8 * KPT) == 0) { f(Int<8>{}); return; } }
        if constexpr (PER_T >= 4) { if (p.page_size % (4 * KPT) == 0) { f(Int<4>{}); return; } }
        if constexpr (PER_T >= 2) { if (p.page_size % (2 * KPT) == 0) { f(Int<2>{}); return; } }
        f(Int<1>{});
    };
    // (of keys that do not exist: some that can be read)
    auto number = [&](int stage, int j, int keys) { return std::min(stage * KT + (wave * PER_T + j) * KPT, p.capacity - keys); };
    auto find = [&](int stage) __attribute__((always_inline)) {
        if constexpr (WHOLE)
            by_runs([&](auto run) __attribute__((always_inline)) {
                constexpr int R = decltype(run)::value;
#pragma unroll
                for (int j = 0; j < PER_T; j += R) next_page[j] = table[tree_column(p, number(stage, j, R * KPT))];
            });
    };
    auto load = [&](int stage, int buffer) __attribute__((always_inline)) {
        if constexpr (WHOLE) {
            by_runs([&](auto run) __attribute__((always_inline)) {
                constexpr int R = decltype(run)::value, N = R < 4 ? R : 4;
#pragma unroll
                for (int j = 0; j < PER_T; j += R) {
                    const int first_key = number(stage, j, R * KPT);
                    const int64_t from = from_page(next_page[j], first_key - tree_column(p, first_key) * p.page_size);
                    const uint32_t to = lds0 + (uint32_t)(buffer * STAGE + (wave * PER_T + j) * 1024);
#pragma unroll
                    for (int i = 0; i < R; i += N) {
                        run_to_lds<N>(K + from + i * 1024, offset + j + i, to + i * 1024);
                        run_to_lds<N>(V + from + i * 1024, offset + j + i, to + i * 1024 + HALF);
                    }
                }
            });
        } else {
            int page[PER_T], row[PER_T];
#pragma unroll
            for (int j = 0; j < PER_T; ++j) {
                const int key = std::min(stage * KT + (wave * PER_T + j) * KPT + lane / Tile::PIECES, p.capacity - 1), column = tree_column(p, key);
                page[j] = columns[column];
                row[j] = key - column * p.page_size;
            }
            char* to = reinterpret_cast<char*>(lds) + buffer * STAGE + wave * PER_T * 1024 + lane * 16;
#pragma unroll
            for (int j = 0; j < PER_T; ++j) {
                const int64_t from = from_page(page[j], row[j]) + (offset[j] - lane / Tile::PIECES * Tile::ROW);
                const Piece k = *reinterpret_cast<const Piece*>(K + from), v = *reinterpret_cast<const Piece*>(V + from);
                *reinterpret_cast<Piece*>(to + j * 1024) = k;
                *reinterpret_cast<Piece*>(to + j * 1024 + HALF) = v;
            }
        }
    };

    if (count > 0) find(last - 1);
#pragma unroll
    for (int s = 0; s < NS - 1; ++s)
        if (s < count) {
            load(last - 1 - s, s);
            if (s + 1 < count) find(last - 2 - s);
        }

    // ---- queries: row r of a slice is head r % share of token r / share --------------------------------
    const int64_t row = row0 + n, known_row = row < rows ? row : rows - 1;
    const int token = (int)(known_row / p.share);
    int ancestor = token;
    Operand<T> q[Wave::QP];
    const T* query = static_cast<const T*>(p.q) + ((b * p.tokens + token) * p.heads + group * p.share + (int)(known_row % p.share)) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < Wave::QP; ++s) {
        T v[8];
#pragma unroll
        for (int j = 0; j < 8 / E; ++j) {
            const Piece piece = *reinterpret_cast<const UnalignedPiece*>(query + 16 * s + j * E);
#pragma unroll
            for (int e = 0; e < E; ++e) v[j * E + e] = piece[e];
        }
        q[s].set(v);
    }
    // The queries are here before the loop begins: the compiler would wait for them in it, each time, and so for all transfers, which count with them.
#pragma unroll
    for (int s = 0; s < Wave::QP; ++s)
        if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(q[s].part[0]));
    f32x16 out[VT];
    float base = -__builtin_inff(), sum = 0.0f, lost = 0.0f;   // of the scores times scale_log2; the lane's share of the sum, and what it lost by rounding (float32)
#pragma unroll
    for (int c = 0; c < VT; ++c) out[c] = f32x16{};

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
                const int at = tid + j * NT, key = at / Tile::PIECES;   // (any share of the stage)
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
        if (stage * KT + key_wave * SUB * 32 >= wave_end) continue;   // (the same for the wave)
        // The scores of the next 32 keys are taken between the powers of these, their maxima between the products with the values of these.
        f32x16 scores[SUB];
        const uint32_t keys0 = lds0 + (uint32_t)(buffer * STAGE + key_wave * SUB * 32 * Tile::ROW);
        constexpr int QP = Wave::QP, BATCH = QP < 8 ? QP : 8;
        typename Values<T, 8>::vec kh[AHEAD ? BATCH : 1];
        auto key_place = [&](int u) __attribute__((always_inline)) {
            uint32_t lds_k = keys0 + (uint32_t)(u * 32 * Tile::ROW) + key_at;
            asm volatile("" : "+v"(lds_k));   // (nothing made of it is kept from one pass to the next)
            return lds_k;
        };
        if constexpr (AHEAD) {
            const uint32_t at = key_place(SUB - 1);
            tree_read_keys<T, D, BATCH>(at, 0, kh);
            __builtin_amdgcn_sched_barrier(0);
            tree_scores<T, D, BATCH>(at, kh, q, scores[SUB - 1], [](int) {});
        } else tree_scores_f32<D>(key_place(SUB - 1), q, scores[SUB - 1]);
        float largest;   // of the lane's scores of 32 keys
        auto look = [&](int u, int r0, int r1) __attribute__((always_inline)) {
#pragma unroll
            for (int r = r0; r < r1; ++r) largest = r ? fmaxf(largest, scores[u][r]) : scores[u][0];
        };
        look(SUB - 1, 0, 16);
#pragma unroll
        for (int u = SUB - 1; u >= 0; --u) {
            const int local = (key_wave * SUB + u) * 32, key0 = stage * KT + local;
            uint32_t lds_v = keys0 + (uint32_t)(u * 32 * Tile::ROW) + HALF + value_at;
            asm volatile("" : "+v"(lds_v));
            uint32_t next_k = 0;
            typename Values<T, 8>::vec held[AHEAD ? 2 * VT : 1];
            f32x16& s = scores[u];
            if constexpr (AHEAD) {
                if (u > 0) {
                    next_k = key_place(u - 1);
                    tree_read_keys<T, D, BATCH>(next_k, 0, kh);
                }
                tree_read_values<T, D, VT>(lds_v, held);
                __builtin_amdgcn_sched_barrier(0);
            } else if (u > 0) tree_scores_f32<D>(key_place(u - 1), q, scores[u - 1]);
            uint32_t seen = ~0u;   // of the 32 keys
            if (key0 + 32 > wave_all) {
                if (p.parents) {
                    seen = lowest_bits(length - key0);
                    while (length + ancestor >= key0 && ancestor >= 0) {
                        const int bit = length + ancestor - key0;
                        if (bit < 32) seen |= 1u << bit;
                        ancestor = parents[ancestor];
                    }
                } else {
                    seen = lowest_bits(length - key0 + token + 1);   // (in this order no sum leaves 32 bits)
                }
                seen &= lowest_bits(total - key0);
                const uint32_t mine = seen >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!(mine >> (8 * (r / 4) + r % 4) & 1)) s[r] = -__builtin_inff();
                look(u, 0, 16);
            }
            // The base of a row's powers is the largest score so far, or up to 8 below it: P is at most 2^8, and outputs are rarely scaled. float16 has no
            // values below 2^-25 and few digits below 2^-14, where many keys of little weight may outweigh the rest: 10 to 15 below the largest score.
            constexpr float BELOW = std::is_same_v<T, f16> ? 10.0f : 0.0f, MOST = std::is_same_v<T, f16> ? 15.0f : 8.0f;
            const float m = across_halves(largest, [](float x, float y) { return fmaxf(x, y); }) * p.scale_log2;
            if (__any(m > base + MOST)) {
                const float now = fmaxf(base, m - BELOW), factor = base == now ? 1.0f : __builtin_amdgcn_exp2f(base - now);
                base = now;
                sum *= factor;
                lost *= factor;
#pragma unroll
                for (int c = 0; c < VT; ++c) out[c] *= factor;
            }
            const float from = base == -__builtin_inff() ? 0.0f : base;   // no key so far: exp2(-inf)
            auto powers = [&](int r0, int r1) __attribute__((always_inline)) {
#pragma unroll
                for (int r = r0; r < r1; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], p.scale_log2, -from));
            };
            if constexpr (AHEAD) {
                // Vector instructions in between of the products, a few to each: a wave's own hide there almost whole, those of the SIMD's other wave do not. By two waves to a SIMD, in a kernel
                // of nothing else: products with two powers and two multiply-adds behind each take 9 % longer than without, with seven multiply-adds 3 %; a wave's products beside another wave's
                // multiply-adds, as many as take the same time alone, 35 %.
                constexpr int EACH = 16 / QP, LATER = 8 / VT;   // powers to a product, the maxima as many as LATER
                __builtin_amdgcn_sched_barrier(0);
                if (u > 0) {
                    tree_scores<T, D, BATCH>(next_k, kh, q, scores[u - 1], [&](int n) __attribute__((always_inline)) {
                        powers(n * EACH, (n + 1) * EACH);
                        __builtin_amdgcn_sched_barrier(0);
                    });
                    tree_values<T, VT>(held, s, out, sum, [&](int n) __attribute__((always_inline)) {
                        look(u - 1, n * LATER, (n + 1) * LATER);
                        asm volatile("" : "+v"(largest));   // (taken here, not where it is needed)
                        __builtin_amdgcn_sched_barrier(0);
                    });
                } else {
                    powers(0, 8);
                    tree_values<T, VT>(held, s, out, sum, [&](int n) __attribute__((always_inline)) {
                        if (n < VT) {
                            powers(8 + n * LATER, 8 + (n + 1) * LATER);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    });
                }
            } else {
                powers(0, 16);
                tree_values_f32<D, VT>(lds_v, s, out, sum, lost);
                if (u > 0) look(u - 1, 0, 16);
            }
            if (!odd) continue;
            for (uint32_t left = __builtin_amdgcn_readfirstlane(odd[local / 32]); left; left &= left - 1) {
                const int key = __builtin_ctz(left), at = key0 + key, column = tree_column(p, at);
                const T* value = reinterpret_cast<const T*>(V + from_page(columns[column], at - column * p.page_size));
                float weight = 0.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r) weight = r == key / 8 * 4 + key % 4 ? s[r] : weight;
                weight = __shfl(weight, n + key / 4 % 2 * 32);
                if (!(seen >> key & 1)) continue;
#pragma unroll
                for (int c = 0; c < VT; ++c)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float v = (float)value[32 * (column_wave * VT + c) + 8 * (r / 4) + 4 * h + r % 4];
                        if (!(__builtin_fabsf(v) < __builtin_inff())) out[c][r] += sizeof(T) == 4 ? __builtin_nanf("") : weight * v;   // (float32: as its three parts have it)
                    }
            }
        }
    }
    sum = across_halves(sum + lost, [](float x, float y) { return x + y; });

    // ---- the shares of the keys meet, in pairs ------------------------------------------------------------
    if constexpr (KW > 1) {
        float* exchange = reinterpret_cast<float*>(lds);
        __shared__ float base_sum[KW][RW][2][32];
        __syncthreads();   // nobody reads the stages any more
        if (h == 0 && column_wave == 0) {   // (the others have the same)
            base_sum[key_wave][row_wave][0][n] = base;
            base_sum[key_wave][row_wave][1][n] = sum;
        }
        __syncthreads();
        float top = -__builtin_inff(), whole_sum = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; ++w) top = fmaxf(top, base_sum[w][row_wave][0][n]);
        const float from = top == -__builtin_inff() ? 0.0f : top, factor = __builtin_amdgcn_exp2f(base - from);
#pragma unroll
        for (int w = 0; w < KW; ++w) whole_sum = fmaf(base_sum[w][row_wave][1][n], __builtin_amdgcn_exp2f(base_sum[w][row_wave][0][n] - from), whole_sum);
        base = top;
        sum = whole_sum;
#pragma unroll
        for (int c = 0; c < VT; ++c) out[c] *= factor;
#pragma unroll
        for (int step = KW / 2; step >= 1; step /= 2) {
            float* const slot = exchange + (((key_wave % step) * CW + column_wave) * RW + row_wave) * EXCHANGE;
            if (key_wave >= step && key_wave < 2 * step) {
#pragma unroll
                for (int c = 0; c < VT; ++c)
#pragma unroll
                    for (int r = 0; r < 16; ++r) slot[(16 * c + r) * WAVE + lane] = out[c][r];
            }
            __syncthreads();
            if (key_wave < step) {
#pragma unroll
                for (int c = 0; c < VT; ++c)
#pragma unroll
                    for (int r = 0; r < 16; ++r) out[c][r] += slot[(16 * c + r) * WAVE + lane];
            }
            __syncthreads();
        }
    }

    if (key_wave || row >= rows) return;
    if (parts > 1) {
        const int64_t at = (int64_t)blockIdx.x * p.block_rows + (row - block * ROWS);
        if (h == 0 && column_wave == 0) {
            p.partial_ml[2 * at] = base;
            p.partial_ml[2 * at + 1] = sum;
        }
#pragma unroll
        for (int c = 0; c < VT; ++c)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(p.partial_o + at * D + 32 * (column_wave * VT + c) + 8 * g + 4 * h) =
                    f32x4{out[c][4 * g], out[c][4 * g + 1], out[c][4 * g + 2], out[c][4 * g + 3]};
        return;
    }
    const float factor = sum == 0.0f ? tree_no_weights(p, entry, token, [&](int at) { return (int)parents[at]; }) : 1.0f / sum;
    T* to = static_cast<T*>(p.o) + ((b * p.tokens + token) * p.heads + group * p.share + (int)(row % p.share)) * D;
#pragma unroll
    for (int c = 0; c < VT; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = out[c][4 * g + e] * factor;
            store_values(to + 32 * (column_wave * VT + c) + 8 * g + 4 * h, o, 4);
        }
}

// The parts of a row joined: WAVES waves to a row share its parts, the lanes of each are the D values. A block of one part is done.
template <class T, int D, int WAVES>
__global__ __launch_bounds__(WAVES < 4 ? 256 : 64 * WAVES) void tree_join_kernel(TreeArgs p) {
    constexpr int PER_LANE = D / WAVE, ROWS = WAVES < 4 ? 4 / WAVES : 1, BATCH = 8;
    __shared__ float sums[ROWS * WAVES][D + 2];
    const int64_t rows = p.tokens * p.share;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), share = wave % WAVES;
    const int64_t at = (int64_t)blockIdx.x * ROWS + wave / WAVES;   // of a slice's row
    if (at >= p.batch * p.kv_heads * rows) return;   // (of waves that share a row: all)
    const int64_t slice = at / rows, row = at % rows, b = slice / p.kv_heads, block = row / p.block_rows;
    const int group = (int)(slice % p.kv_heads);
    const int parts = __builtin_amdgcn_readfirstlane(p.plan[2 * b + 1]);
    if (parts == 1) return;
    T* to = static_cast<T*>(p.o) + ((b * p.tokens + row / p.share) * p.heads + group * p.share + (int)(row % p.share)) * D + lane * PER_LANE;
    float top = -__builtin_inff(), sum = 0.0f, o[PER_LANE] = {};
    const int64_t first = p.plan[2 * b] + (group * p.row_blocks + block) * parts;   // workgroup
    for (int part = share; part < parts; part += BATCH * WAVES) {
        float base[BATCH], weight[BATCH], values[BATCH][PER_LANE], now = top;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const bool real = part + i * WAVES < parts;
            const int64_t from = (first + (real ? part + i * WAVES : part)) * p.block_rows + (row - block * p.block_rows);
            base[i] = real ? p.partial_ml[2 * from] : -__builtin_inff();
            weight[i] = real ? p.partial_ml[2 * from + 1] : 0.0f;
            load_values(values[i], p.partial_o + from * D + lane * PER_LANE, PER_LANE);
            if (!real)
#pragma unroll
                for (int e = 0; e < PER_LANE; ++e) values[i][e] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) now = fmaxf(now, base[i]);
        const float from = now == -__builtin_inff() ? 0.0f : now, factor = __builtin_amdgcn_exp2f(top - from);
        sum *= factor;
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) o[e] *= factor;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const float f = __builtin_amdgcn_exp2f(base[i] - from);
            sum = fmaf(weight[i], f, sum);
#pragma unroll
            for (int e = 0; e < PER_LANE; ++e) o[e] = fmaf(values[i][e], f, o[e]);
        }
        top = now;
    }
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) sums[wave][lane * PER_LANE + e] = o[e];
        if (lane == 0) sums[wave][D] = top, sums[wave][D + 1] = sum;
        __syncthreads();
        if (share) return;
        float all = top;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) all = fmaxf(all, sums[wave + w][D]);
        const float from = all == -__builtin_inff() ? 0.0f : all, factor = __builtin_amdgcn_exp2f(top - from);
        sum *= factor;
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) o[e] *= factor;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(sums[wave + w][D] - from);
            sum = fmaf(sums[wave + w][D + 1], f, sum);
#pragma unroll
            for (int e = 0; e < PER_LANE; ++e) o[e] = fmaf(sums[wave + w][lane * PER_LANE + e], f, o[e]);
        }
    }
    const float scale = sum == 0.0f ? tree_no_weights(p, tree_entry(p, b), (int)(row / p.share), [&](int at) { return p.parents[b * p.tokens + at]; }) : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < PER_LANE; ++e) o[e] *= scale;
    store_values(to, o, PER_LANE);
}

// PAIR: 64 rows by two row and two key waves, two workgroups to a CU; DEEP: 64 rows by two and four, one to a CU; TALL: 128 rows by four row waves, two to a CU, where each SIMD has two waves
// and the matrix unit is busy, but with one to a CU it has one. Heads of more than 256 bytes: one to a CU, no DEEP. (32 rows by two waves were behind PAIR with few rows too:
// two waves are not enough to get the transfers out.)
enum { TREE_PAIR, TREE_DEEP, TREE_TALL, TREE_FORMS };

// us: of 64 keys where a workgroup has its CU alone, and where another shares it; of a row of workgroups besides
struct TreeForm { int rows, places; double alone, shared, start; };
static TreeForm tree_form(int form, int bytes, bool f32) {
    const int size = bytes / (f32 ? 4 : 2);
    // as they fit the times of calls in all forms: 1 to 128 entries of 1 to 4096 tokens behind 0 to 16000, 1 to 16 heads to a group
    const double rates[6][TREE_FORMS][2] = {{{0.55, 0.8}, {0.4, 0.4}, {0.8, 2.0}},      // 16 bits, heads of 64
                                            {{0.85, 1.4}, {0.7, 0.7}, {1.05, 1.65}},    // 128
                                            {{1.45, 1.45}, {}, {1.95, 1.95}},           // 256
                                            {{1.75, 1.95}, {1.45, 1.45}, {2.95, 4.0}},  // float32, 64
                                            {{3.2, 3.2}, {}, {4.6, 4.6}},
                                            {{7.6, 7.6}, {}, {8.2, 8.2}}};
    const double(&rate)[2] = rates[(f32 ? 3 : 0) + (size == 64 ? 0 : size == 128 ? 1 : 2)][form];
    return {form == TREE_TALL ? 128 : 64, form == TREE_DEEP || bytes > 256 ? 256 : 512, rate[0], rate[1], form == TREE_DEEP ? 9.0 : 8.0};
}

// How a call is cut: which form, and how many workgroups the parts of its blocks are dealt to (0: one to a block), by what the forms take if the longest of the entries fills its table and they do
// by two thirds. Measured, us, at heads of 128 in 16 bits, 32 heads in 8 groups (PAIR / DEEP / TALL, one workgroup to a block; the same in parts): 16 x 1 token of up to 8192 147 / 120 / 174,
// 73 / 80 / 91; 32 x 1 of 8000 156 / 139 / 168, 129 / 142 / 172; 8 trees of 64 behind 1400 to 3000 54 / 43 / 73, 67 / 60 / 59; 2 of 256 behind 1600 to 2700 54 / 42 / 75, 56 / 48 / 62; 4 of 32 behind
// 1400 to 3800 61 / 48 / 87, 30 / 30 / 28; a prompt of 512 14.5 / 14.6 / 18, 30 / 21 / 30; of 1024 24 / 33 / 30, 36 / 24 / 38; of 2048 57 / 75 / 53, 54 / 54 / 53; 4096 behind 4096, 16 heads in 4 groups,
// 235 / 269 / 214, 234. Over 70 calls of drawn sizes, all types and head sizes, in tables that fit, the choice takes 1 % more than the least of all forms for half of them, 5 % on average, and up to
// 1.5 times as long (99 x 2162 tokens behind up to 2600, 2 heads of 64: PAIR 679, TALL 457).
// A table with more columns than the lengths take is priced as if they were filled. With columns for 131072 keys the same 70 calls take 22 % more than the least on average, 30 of them 2 to 5 us for parts
// that short caches do not need, 1.7 times as long at most; 8 trees of 64 57 for 42, 2 of 256 61 for 42, a prompt of 1024 30 for 24. One token for each of 16 to 300 entries and prompts from 2048 on are
// as they were.
struct TreeCut { int form, block_rows, dealt; int64_t row_blocks; };
static TreeCut tree_cut(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t capacity, int64_t size, int type) {
    const bool f32 = type == MI355X_TYPE_FLOAT;
    const int bytes = (int)size * (f32 ? 4 : 2), forced = tuning().tree_form, wanted = tuning().tree_deal;
    const int64_t rows = tokens * (heads / kv_heads), slices = batch * kv_heads;
    const double most = std::max(1.0, (double)capacity / 64), mean = std::max(1.0, ((double)capacity - 0.5 * (double)std::min(tokens, capacity)) / 64);
    const double full = batch > 1 ? 0.67 : 1.0, least_memory = full * (double)slices * (double)capacity * 2 * bytes / 5e6;
    TreeCut best = {};
    double least = __builtin_inf();
    for (int form = 0; form < TREE_FORMS; ++form) {
        if ((forced >= 0 && forced < TREE_FORMS && form != forced) || (form == TREE_DEEP && bytes > 256)) continue;
        const TreeForm f = tree_form(form, bytes, f32);
        const int64_t blocks = ceil_div(rows, (int64_t)f.rows), items = blocks * slices;
        const int block_rows = (int)std::min<int64_t>(f.rows, rows);
        // what the bytes take goes by how many workgroups ask for them, and a little by how often; with one to a block the longest entry's are the last
        const double memory = least_memory * (form == TREE_DEEP ? 0.95 : 0.7) * (1 + 0.08 * (double)(blocks - 1)), uneven = batch > 1 ? 1.25 : 1.0, rounds = (double)items / f.places;
        const double whole = f.start + std::max(memory * uneven, items <= 256 ? most * f.alone : items <= f.places ? std::max(most * f.alone, full * mean * f.shared) :
                                                                  rounds * full * mean * (f.places > 256 ? f.shared : f.alone) + (rounds - 1) * f.start);
        if (wanted <= 0 && whole < least) least = whole, best = {form, block_rows, 0, blocks};
        const int64_t places = wanted > 0 ? wanted : form == TREE_TALL ? 256 : f.places;
        if (wanted == 0 || items > places || batch > DEAL_ENTRIES) continue;
        // parts are whole stages, and no block has less than one; 5.5 for finding them and for the join, and 2e-6 for a value that goes through memory
        const double used = std::min((double)places, (double)items * most);
        const double parts = f.start + 5.5 + std::max(memory, 1.7 * (double)items * full * most / used * (used > 256 ? f.shared : f.alone)) + used * block_rows * (double)size * 2e-6;
        if (parts < least) least = parts, best = {form, block_rows, (int)places, blocks};
    }
    if (!best.row_blocks) {   // (forced, and not possible so)
        const TreeForm f = tree_form(TREE_PAIR, bytes, f32);
        best = {TREE_PAIR, (int)std::min<int64_t>(f.rows, rows), 0, ceil_div(rows, (int64_t)f.rows)};
    }
    return best;
}

static int64_t tree_scratch(const TreeCut& cut, int64_t batch, int64_t size) { return cut.dealt ? (int64_t)cut.dealt * cut.block_rows * (size + 2) + 2 * batch : 0; }

template <class T, int D>
static int launch_tree(TreeArgs p, const TreeCut& cut, hipStream_t st) {
    constexpr int BYTES = D * (int)sizeof(T);
    const int64_t rows = p.tokens * p.share, slices = p.batch * p.kv_heads;
    bool fits = true;
    auto launch = [&](auto rw, auto cw, auto kw, auto sub, auto ns, auto per_simd) {
        constexpr int RW = decltype(rw)::value, CW = decltype(cw)::value, KW = decltype(kw)::value, SUB = decltype(sub)::value, NS = decltype(ns)::value;
        constexpr int PER_SIMD = decltype(per_simd)::value;
        const int64_t grid = p.dealt ? p.dealt : p.row_blocks * slices;
        // A wave has eight parts of a row on their way at once: four and sixteen waves to a row of more. us by four / sixteen: 16 rows of 128 parts 5.8 / 5.0, 32 of 64 3.9 / 4.5.
        const int64_t parts = p.dealt / (p.row_blocks * slices);
        const int join_waves = parts > 64 ? 16 : parts > 16 ? 4 : 1;
        const int64_t joins = p.dealt ? join_waves > 1 ? slices * rows : ceil_div(slices * rows, (int64_t)4) : 0;
        fits = grid_fits(grid, 64 * RW * CW * KW) && grid_fits(joins, 1024);
        if (!fits) return;
        const dim3 g((unsigned)grid), threads(64 * RW * CW * KW);
        if (p.page_size % (1024 / BYTES) == 0) hipLaunchKernelGGL((tree_attention_kernel<T, D, RW, CW, KW, SUB, NS, PER_SIMD, true>), g, threads, 0, st, p);
        else hipLaunchKernelGGL((tree_attention_kernel<T, D, RW, CW, KW, SUB, NS, PER_SIMD, false>), g, threads, 0, st, p);
        if (!joins) return;
        if (join_waves == 16) hipLaunchKernelGGL((tree_join_kernel<T, D, 16>), dim3((unsigned)joins), dim3(1024), 0, st, p);
        else if (join_waves == 4) hipLaunchKernelGGL((tree_join_kernel<T, D, 4>), dim3((unsigned)joins), dim3(256), 0, st, p);
        else hipLaunchKernelGGL((tree_join_kernel<T, D, 1>), dim3((unsigned)joins), dim3(256), 0, st, p);
    };
    // Heads of 256: a wave with all of their columns has no room for its sums beside the queries (they move between two register files for every 32 keys), two with half of them each have it,
    // and take the scores twice. us, 4 x 64 tokens behind 4096, 16 heads in 4 groups: bfloat16 128 -> 109, 128 rows a workgroup 214 -> 178, float32 939 -> 693; float32 heads of 128 are behind so.
    constexpr bool WIDE = BYTES > 256, WIDEST = BYTES > 512;
    constexpr int CW = D == 256 ? 2 : 1, PER_SIMD = WIDE && (D != 256 || WIDEST) ? 1 : 2;
    if (cut.form == TREE_PAIR) launch(Int<2>{}, Int<CW>{}, Int<(WIDEST ? 1 : 2)>{}, Int<1>{}, Int<(BYTES == 128 ? 4 : 2)>{}, Int<PER_SIMD>{});
    else if (cut.form == TREE_TALL) launch(Int<4>{}, Int<(WIDEST ? 1 : CW)>{}, Int<1>{}, Int<(WIDE ? 1 : 2)>{}, Int<2>{}, Int<PER_SIMD>{});
    else if constexpr (!WIDE) launch(Int<2>{}, Int<1>{}, Int<4>{}, Int<1>{}, Int<(BYTES == 128 ? 4 : 2)>{}, Int<2>{});
    MI355X_REQUIRE(fits, "tree_attention: too large");
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
    return batch && tokens && heads ? tree_scratch(tree_cut(batch, tokens, heads, kv_heads, page_size * columns, size, type), batch, size) : 0;
}

extern "C" int mi355x_tree_attention(const void* Q, const void* k_pages, const void* v_pages, const int32_t* table, const int32_t* lengths, const int32_t* parents, void* O,
                                     float* scratch, int64_t scratch_floats, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t size, int64_t pages,
                                     int64_t page_size, int64_t columns, float scale, int type, void* stream) {
    using namespace mi355x;
    MI355X_REQUIRE(is_mixed_type(type), "tree_attention: element type %d", type);
    MI355X_REQUIRE(size == 64 || size == 128 || size == 256, "tree_attention: head size %lld (64, 128 and 256 are supported)", (long long)size);
    MI355X_REQUIRE(heads >= 0 && kv_heads >= 1 && heads % kv_heads == 0, "tree_attention: %lld heads share keys and values in %lld groups", (long long)heads, (long long)kv_heads);
    MI355X_REQUIRE(scale > 0.0f && scale * LOG2_E < __builtin_inff(), "tree_attention: scale %g (a positive number is needed)", (double)scale);
    MI355X_REQUIRE(!parents || tokens <= TREE_MOST, "tree_attention: a tree of %lld tokens (%d at most)", (long long)tokens, TREE_MOST);
    MI355X_REQUIRE(tree_fits(batch, tokens, heads, kv_heads, size, page_size, columns) && pages >= 1 && pages < (int64_t)1 << 31 &&
                       (double)pages * page_size * kv_heads < 0x1p46, "tree_attention: negative, empty or too large an extent");
    if (batch == 0 || tokens == 0 || heads == 0) return MI355X_OK;
    MI355X_REQUIRE(Q && O && k_pages && v_pages && lengths && (columns == 0 || table), "tree_attention: null pointer");
    MI355X_REQUIRE(((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) == 0, "tree_attention: pages have to stand at 16-byte boundaries");
    const TreeCut cut = tree_cut(batch, tokens, heads, kv_heads, page_size * columns, size, type);
    const int64_t floats = tree_scratch(cut, batch, size);
    MI355X_REQUIRE(floats == 0 || (scratch && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0 && scratch_floats >= floats), "tree_attention: scratch memory for %lld floats, 16-byte aligned",
                   (long long)floats);
    TreeArgs p = {};
    p.q = Q; p.k_pages = k_pages; p.v_pages = v_pages; p.table = table; p.lengths = lengths; p.parents = parents; p.o = O;
    p.partial_o = scratch;
    p.partial_ml = scratch ? scratch + (int64_t)cut.dealt * cut.block_rows * size : nullptr;
    p.plan = scratch ? reinterpret_cast<int32_t*>(p.partial_ml + (int64_t)2 * cut.dealt * cut.block_rows) : nullptr;
    p.batch = batch; p.tokens = tokens; p.columns = columns; p.row_blocks = cut.row_blocks; p.block_rows = cut.block_rows; p.dealt = cut.dealt;
    p.order = cut.row_blocks * batch * kv_heads <= 512;
    p.pages = (int)pages; p.page_size = (int)page_size; p.capacity = (int)(page_size * columns);
    p.heads = (int)heads; p.kv_heads = (int)kv_heads; p.share = (int)(heads / kv_heads);
    while (((int64_t)1 << p.page_shift) < page_size) ++p.page_shift;
    p.page_magic = (uint32_t)((((uint64_t)1 << (31 + p.page_shift)) + (uint64_t)page_size - 1) / (uint64_t)page_size);
    p.scale_log2 = scale * LOG2_E;
    int status = MI355X_OK;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        hipStream_t st = static_cast<hipStream_t>(stream);
        status = size == 64 ? launch_tree<T, 64>(p, cut, st) : size == 128 ? launch_tree<T, 128>(p, cut, st) : launch_tree<T, 256>(p, cut, st);
    });
    return status;
}
