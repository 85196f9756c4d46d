// QuantizedLinear: Y = act(xs[m] ws[n] sum_k X[m,k] W[n,k] + b[n]) + R[m,n]; X and W in int8, both k-contiguous (W as a linear layer keeps it), Y, b
// and R in float32, float16 or bfloat16. The sums are int32 and exact (K below 2^17), everything behind them float32, rounded once. The reference has
// no such node: it runs MatMulInteger, a Cast, two Muls and the rest one after the other.
// Bound by the matrix unit in tiles: 8192 x 8192 x 4096 256 us (2.15 POP/s; the vendor's int8 product alone 258 to 271, 2.03 to 2.13), of which the results' way out is 43;
// its loop runs at 2.6 POP/s, where the operands' reads from LDS (six of 1 KB for eight products of a wave) take as long as the products. Few rows by the
// weights' way in: 4 x 4096 x 4096 6.1 us, 2.7 TB/s, of which 3.5 do not depend on the size.
#include "mixed.h"
#include "gemm_tile.h"

#include <algorithm>

namespace mi355x {

struct QLinArgs {
    const int8_t* X; const int8_t* W; const float* xs; const float* ws;
    const void* bias; const void* residual; void* Y;
    int64_t M, N, K;
    int xs_step, ws_step;   // 0: one scale for all
    int activation;
    int64_t tiles_m, tiles_n;
};

// NaN stays NaN. Silu of 16-bit results with one reciprocal and one power of two, off by |v| 2^-24 of the result where v is negative: 2^-17 at most before it vanishes.
// float32 results by the library's exponential and a division.
template <class T, int ACT>
__device__ __forceinline__ float activated(float v) {
    if (ACT == MI355X_ACT_RELU) return v < 0.0f ? 0.0f : v;
    if (ACT == MI355X_ACT_GELU) return gelu_erf(v);
    if (ACT == MI355X_ACT_SILU && std::is_same_v<T, float>) return v / (1.0f + expf(-v));
    if (ACT == MI355X_ACT_SILU) return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
    return v;
}

// The epilogue of R rows that a lane has four results next to each other of, in each of G groups: what it reads first, all at once, because stores hold
// back reads that come after them (the residual may be Y itself). row(r), column(g): where; acc(r, g, e): the sums.
template <class T, int ACT, int R, int G, class Row, class Column, class Sum>
__device__ __forceinline__ void qlin_store(const QLinArgs& p, Row&& row, Column&& column, Sum&& acc) {
    float xs[R], ws[G][4], b[G][4], res[R][G][4];
#pragma unroll
    for (int r = 0; r < R; ++r) xs[r] = p.xs[(row(r) < p.M ? row(r) : p.M - 1) * p.xs_step];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        if (p.ws_step) load_values(ws[g], p.ws + column(g), p.N - column(g));
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) ws[g][e] = p.ws[0];
        if (p.bias) load_values(b[g], static_cast<const T*>(p.bias) + column(g), p.N - column(g));
        if (p.residual) {
#pragma unroll
            for (int r = 0; r < R; ++r) load_values(res[r][g], static_cast<const T*>(p.residual) + row(r) * p.N + column(g), row(r) < p.M ? p.N - column(g) : 0);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = (float)acc(r, g, e) * xs[r] * ws[g][e];
                if (p.bias) v[e] += b[g][e];
                v[e] = activated<T, ACT>(v[e]);
                if (p.residual) v[e] += res[r][g][e];
            }
            store_values(static_cast<T*>(p.Y) + row(r) * p.N + column(g), v, row(r) < p.M ? p.N - column(g) : 0);
        }
}

typedef i32x4 UnalignedBytes __attribute__((aligned(1)));

// The 16 bytes from p on by the aligned words that hold them: 16-byte accesses at other boundaries than those of words take the memory unit up to four times
// as long (64 x 4097 x 4095 straight from memory: 58 us, so 27; 19 with K = 4092). What is read lies between p - 3 and p + 19; the
// bytes before p are the array's own, as that begins at a word.
__device__ __forceinline__ i32x4 words_at(const int8_t* p) {
    typedef i32x4 AtWord __attribute__((aligned(4)));
    const uint32_t bytes = (uint32_t)reinterpret_cast<uintptr_t>(p) & 3;
    const int8_t* first = p - bytes;
    const i32x4 w = *reinterpret_cast<const AtWord*>(first);
    const int next = *reinterpret_cast<const int*>(first + (bytes ? 16 : 12));
    i32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (int)__builtin_amdgcn_alignbyte((uint32_t)(i < 3 ? w[i + 1] : next), (uint32_t)w[i], bytes);
    return v;
}

// the 16 bytes from p on of which `left` belong to a row of K: the others as 0
template <bool WORDS>
__device__ __forceinline__ i32x4 row_bytes(const int8_t* p, int64_t left, int64_t K) {
    if (WORDS && left >= 19) return words_at(p);
    if (left >= 16) return *reinterpret_cast<const UnalignedBytes*>(p);
    if (left <= 0) return i32x4{};
    if (K < 16) {
        int8_t b[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = i < left ? p[i] : (int8_t)0;
        return __builtin_bit_cast(i32x4, b);
    }
    // the row's last 16 bytes, moved down
    typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
    u64x2 v = __builtin_bit_cast(u64x2, *reinterpret_cast<const UnalignedBytes*>(p - (16 - left)));
    const int bits = 8 * (16 - (int)left);   // 8 to 120
    v = bits >= 64 ? u64x2{v.y >> (bits - 64), 0} : u64x2{v.x >> bits | v.y << (64 - bits), v.y >> bits};
    return __builtin_bit_cast(i32x4, v);
}

// Any shape and alignment, operands straight from memory. A workgroup has 16 columns and 16 MT rows of Y, its eight waves take turns at the
// 128-byte lines of K and their sums meet in LDS. WORDS: rows at addresses that are no multiples of 4, in arrays that are, by aligned words.
template <class T, int ACT, int MT, bool WORDS>
__global__ __launch_bounds__(512) void qlin_direct_kernel(QLinArgs p) {
    constexpr int WAVES = 8;
    __shared__ __attribute__((aligned(16))) i32x4 part[WAVES][MT][WAVE];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, l16 = lane % 16, lq = lane / 16;
    const int64_t n0 = (int64_t)blockIdx.x % p.tiles_n * 16, m0 = (int64_t)blockIdx.x / p.tiles_n * 16 * MT;
    const int8_t* w = p.W + std::min(n0 + l16, p.N - 1) * p.K;
    const int8_t* x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = p.X + std::min(m0 + 16 * t + l16, p.M - 1) * p.K;
    i32x4 acc[MT] = {};
    auto line = [&](int64_t k, auto&& bytes) __attribute__((always_inline)) {
        i32x4 a[2], b[2][MT];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int64_t at = k + 64 * s + 16 * lq;
            a[s] = bytes(w + at, p.K - at);
#pragma unroll
            for (int t = 0; t < MT; ++t) b[s][t] = bytes(x[t] + at, p.K - at);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s], b[s][t], acc[t], 0, 0, 0);
    };
    int64_t k = 128 * wave;
#pragma unroll 4
    for (; k + (WORDS ? 131 : 128) <= p.K; k += 128 * WAVES)
        line(k, [](const int8_t* at, int64_t) {
            if constexpr (WORDS) return words_at(at);
            else return i32x4(*reinterpret_cast<const UnalignedBytes*>(at));
        });
    if (k < p.K) line(k, [&](const int8_t* at, int64_t left) { return row_bytes<WORDS>(at, left, p.K); });
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave >= MT) return;
    i32x4 sum = part[0][wave][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += part[w][wave][lane];
    qlin_store<T, ACT, 1, 1>(p, [&](int) { return m0 + 16 * wave + l16; }, [&](int) { return n0 + 4 * lq; }, [&](int, int, int e) { return sum[e]; });
}

// 16 bytes to a lane from global memory, base + the lane's offset, into LDS at lds + 16 lane; base and lds are the same for the wave, all 16-byte aligned.
// Written as assembly because the compiler waits for every builtin transfer before the next LDS read.
__device__ __forceinline__ void qlin_to_lds(const int8_t* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(offset), "s"(base) : "memory", "m0");
}

// What the lanes of a wave wrote to LDS before is read by the others after it, and the other way round. LDS operations of a wave complete in order, so this takes no
// instruction: it keeps the compiler, which sees the addresses of one lane, from moving one across the other.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// Tiles through LDS: WM x WN waves of 32 TM rows and 32 TN columns each, steps of 128 k, NS stages. A row's 128 bytes of a step are eight
// pieces of 16; piece c of row r lies at c ^ (r / 2 % 8), so that the 16 rows whose
// pieces are read at a time lie in 16 different places of the 256 bytes that the banks hold. DIRECT (rows at
// 16-byte boundaries): whole steps go from memory to LDS without registers, NS - 1 steps ahead; otherwise, two
// steps ahead, and for a last part of a step, through registers.
template <class T, int ACT, int WM, int WN, int TM, int TN, int NS, int BK, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void qlin_tile_kernel(QLinArgs p, int group_m) {
    constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, STAGE = (BM + BN) * BK;
    constexpr int PPR = BK / 16, RPT = 64 / PPR;   // pieces of a row, rows of a transfer (1 KB)
    constexpr int PER_WAVE = (BM + BN) / RPT / NW;  // transfers to a wave and step
    static_assert((BM + BN) / RPT % NW == 0 && BM % RPT == 0 && (PPR == 8 || PPR == 16), "whole transfers");
    auto place = [](int row) { return PPR == 8 ? row / 2 % 8 : row % 16; };
    __shared__ __attribute__((aligned(1024))) int8_t lds[NS * STAGE];
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int l32 = lane % 32, h = lane / 32, wm = wave % WM, wn = wave / WM;
    int64_t tm, tn;
    tile_coords(xcd_remap(blockIdx.x, p.tiles_m * p.tiles_n), p.tiles_m, p.tiles_n, group_m, tm, tn);
    const int64_t m0 = tm * BM, n0 = tn * BN;

    // Transfer i of a wave is of X for i below X_COUNT, of W otherwise: a pointer that is the same for the wave and 32 bits of offset to a lane (64 bits to a lane take the
    // memory path several times as long). Rows past the end are the last row again; what they give is not stored.
    constexpr int X_COUNT = BM / RPT / NW;
    static_assert(BM / RPT % NW == 0, "a transfer is of one operand for all waves");
    const int8_t *x_tile = p.X + m0 * p.K, *w_tile = p.W + n0 * p.K;
    uint32_t offset[PER_WAVE];
    int piece[PER_WAVE];
#pragma unroll
    for (int i = 0; i < PER_WAVE; ++i) {
        const int first = RPT * (wave + i * NW), r = (i < X_COUNT ? first : first - BM) + lane / PPR;
        const int64_t left = i < X_COUNT ? p.M - m0 : p.N - n0;
        piece[i] = (lane % PPR) ^ place(first + lane / PPR);
        offset[i] = (uint32_t)((r < left ? r : left - 1) * p.K) + 16u * (uint32_t)piece[i];
    }
    auto base = [&](int i, int64_t step) __attribute__((always_inline)) {
        const uint64_t at = reinterpret_cast<uint64_t>((i < X_COUNT ? x_tile : w_tile) + step * BK);
        return reinterpret_cast<const int8_t*>(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at));
    };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds;
    const int64_t whole = DIRECT ? p.K / BK : 0, steps = (p.K + BK - 1) / BK;
    typedef i32x4 Held[PER_WAVE];
    auto fetch = [&](int64_t step, Held& to) __attribute__((always_inline)) {   // by registers (words and what follows them wait in more of them: 124 us become 190 at 4095^3)
        if ((step + 1) * BK <= p.K) {
#pragma unroll
            for (int i = 0; i < PER_WAVE; ++i) to[i] = *(const __attribute__((address_space(1))) UnalignedBytes*)(base(i, step) + offset[i]);
        } else {
#pragma unroll
            for (int i = 0; i < PER_WAVE; ++i) to[i] = row_bytes<false>((i < X_COUNT ? x_tile : w_tile) + step * BK + offset[i], p.K - step * BK - 16 * piece[i], p.K);
        }
    };
    auto put = [&](int stage, const Held& v) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER_WAVE; ++i) *reinterpret_cast<i32x4*>(lds + stage * STAGE + (wave + i * NW) * 1024 + 16 * lane) = v[i];
    };
    auto load = [&](int64_t step, int stage) __attribute__((always_inline)) {
        if (step < whole) {
#pragma unroll
            for (int i = 0; i < PER_WAVE; ++i) qlin_to_lds(base(i, step), offset[i], lds0 + (uint32_t)(stage * STAGE + (wave + i * NW) * 1024));
        } else if (step < steps) {
            Held part;
            fetch(step, part);
            put(stage, part);
        }
    };

    i32x16 acc[TM][TN] = {};
    auto multiply = [&](int stage, auto&& meanwhile) __attribute__((always_inline)) {
        const int8_t* x = lds + stage * STAGE + (wm * 32 * TM + l32) * BK;
        const int8_t* w = lds + stage * STAGE + (BM + wn * 32 * TN + l32) * BK;
        i32x4 fx[2][TM], fw[2][TN];
        auto read = [&](int set, int ks) __attribute__((always_inline)) {
            const int piece = 16 * ((2 * ks + h) ^ place(l32));
#pragma unroll
            for (int t = 0; t < TN; ++t) fw[set][t] = *reinterpret_cast<const i32x4*>(w + 32 * t * BK + piece);
#pragma unroll
            for (int t = 0; t < TM; ++t) fx[set][t] = *reinterpret_cast<const i32x4*>(x + 32 * t * BK + piece);
        };
        read(0, 0);
        meanwhile();
#pragma unroll
        for (int ks = 0; ks < BK / 32; ++ks) {
            if (ks + 1 < BK / 32) read((ks + 1) % 2, ks + 1);
#pragma unroll
            for (int t = 0; t < TM; ++t)
#pragma unroll
                for (int u = 0; u < TN; ++u) acc[t][u] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[ks % 2][u], fx[ks % 2][t], acc[t][u], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if constexpr (DIRECT) {
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) load(i, i);
        int stage = 0;
        for (int64_t step = 0; step < steps; ++step) {
            // The step is in LDS, and nobody reads any more what the transfer below writes. Transfers complete in order: those of the NS - 2 steps
            // behind this one may be on their way, if they are transfers.
            if (step + NS - 2 < whole) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * PER_WAVE) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __syncthreads();
            multiply(stage, [&] { load(step + NS - 1, stage == 0 ? NS - 1 : stage - 1); });
            stage = stage + 1 == NS ? 0 : stage + 1;
        }
    } else {
        Held held[2];
        if (steps > 0) fetch(0, held[0]);
        if (steps > 1) fetch(1, held[1]);
        for (int64_t step = 0; step < steps; step += 2) {
            static_for<2>([&](auto odd) __attribute__((always_inline)) {
                constexpr int s = decltype(odd)::value;
                if (step + s < steps) {
                    put(s, held[s]);
                    __syncthreads();
                    multiply(s, [&] { if (step + s + 2 < steps) fetch(step + s + 2, held[s]); });
                }
            });
        }
    }
    // The results leave by whole lines: a lane has four neighbours of one row, and of the next instruction's rows others; 32 rows at a time go through LDS, of which
    // each wave has a share of its own, as floats (times the row's scale), and come back as rows. Stored as they lie, 16 bytes of each row at a time, a tile's
    // results took 17 us.
    constexpr int PIECES = 8 * TN, PER_STEP = WAVE / PIECES, COUNT = 32 / PER_STEP;   // pieces of 16 bytes in a row, rows to an instruction
    constexpr int BATCH = COUNT < 8 ? COUNT : 8;
    static_assert(NW * 32 * 32 * TN * 4 <= NS * STAGE, "the waves' shares fit");
    float* mine = reinterpret_cast<float*>(lds) + wave * 32 * 32 * TN;
    auto at = [&](int row, int column) { return row * 32 * TN + 4 * (column / 4 ^ (TN == 1 ? row / 2 % 8 : row % 16)) + column % 4; };
    const int c = 4 * (lane % PIECES);
    const int64_t n = n0 + wn * 32 * TN + c, left = p.N - n;
    float ws[4], bias[4] = {};
    if (p.ws_step) load_values(ws, p.ws + n, left);
    else ws[0] = ws[1] = ws[2] = ws[3] = p.ws[0];
    if (p.bias) load_values(bias, static_cast<const T*>(p.bias) + n, left);
    __syncthreads();   // nobody reads the stages any more
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const int64_t m = m0 + (wm * TM + t) * 32;
        const float xs = p.xs[(m + l32 < p.M ? m + l32 : p.M - 1) * p.xs_step];
#pragma unroll
        for (int u = 0; u < TN; ++u)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(mine + at(l32, 32 * u + 8 * g + 4 * h)) =
                    f32x4{(float)acc[t][u][4 * g] * xs, (float)acc[t][u][4 * g + 1] * xs, (float)acc[t][u][4 * g + 2] * xs, (float)acc[t][u][4 * g + 3] * xs};
        wave_lds_fence();   // lanes read what others wrote
#pragma unroll
        for (int i0 = 0; i0 < COUNT; i0 += BATCH) {
            float res[BATCH][4];
            if (p.residual) {   // all at once: stores hold back reads that come after them, the residual may be Y itself
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int64_t r = m + (i0 + i) * PER_STEP + lane / PIECES;
                    load_values(res[i], static_cast<const T*>(p.residual) + r * p.N + n, r < p.M ? left : 0);
                }
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int row = (i0 + i) * PER_STEP + lane / PIECES;
                const f32x4 sum = *reinterpret_cast<const f32x4*>(mine + at(row, c));
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = activated<T, ACT>(sum[e] * ws[e] + bias[e]);
                    if (p.residual) v[e] += res[i][e];
                }
                store_values(static_cast<T*>(p.Y) + (m + row) * p.N + n, v, m + row < p.M ? left : 0);
            }
        }
        wave_lds_fence();   // the next 32 rows go where others have read
    }
}

// false: more workgroups than a launch has
template <class T, int ACT>
static bool launch_qlin(QLinArgs p, hipStream_t st) {
    bool fits = true;
    const bool words = ((reinterpret_cast<uintptr_t>(p.X) | reinterpret_cast<uintptr_t>(p.W)) & 3) == 0;
    auto direct = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        p.tiles_n = ceil_div(p.N, (int64_t)16);
        p.tiles_m = ceil_div(p.M, (int64_t)(16 * MT));
        fits = grid_fits(p.tiles_m * p.tiles_n, 512);
        if (!fits) return;
        const dim3 grid((unsigned)(p.tiles_m * p.tiles_n)), block(512);
        if (words && p.K % 4) hipLaunchKernelGGL((qlin_direct_kernel<T, ACT, MT, true>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((qlin_direct_kernel<T, ACT, MT, false>), grid, block, 0, st, p);
    };
    const bool aligned = p.K % 16 == 0 && ((reinterpret_cast<uintptr_t>(p.X) | reinterpret_cast<uintptr_t>(p.W)) & 15) == 0;
    auto tile = [&](auto wm, auto wn, auto tm, auto tn, auto ns, auto bk, int per_cu) {
        constexpr int WM = decltype(wm)::value, WN = decltype(wn)::value, TM = decltype(tm)::value, TN = decltype(tn)::value, NS = decltype(ns)::value, BK = decltype(bk)::value;
        p.tiles_m = ceil_div(p.M, (int64_t)(32 * TM * WM));
        p.tiles_n = ceil_div(p.N, (int64_t)(32 * TN * WN));
        const int64_t nwg = p.tiles_m * p.tiles_n;
        fits = grid_fits(nwg, 64 * WM * WN);
        if (!fits) return;
        const int group_m = choose_group_m(p.tiles_m, ceil_div(nwg, (int64_t)NUM_XCD), (int64_t)per_cu * 32, 32 * TM * WM, 32 * TN * WN, p.K);
        const dim3 grid((unsigned)nwg), block(64 * WM * WN);
        if (aligned) hipLaunchKernelGGL((qlin_tile_kernel<T, ACT, WM, WN, TM, TN, NS, BK, true>), grid, block, 0, st, p, group_m);
        else hipLaunchKernelGGL((qlin_tile_kernel<T, ACT, WM, WN, TM, TN, 2, BK, false>), grid, block, 0, st, p, group_m);
    };
    // Which kernel, by microseconds of the forms at N = K = 4096, bfloat16 (M; 16 columns each direct / 64 x 64 / 128 x 128 one to a CU / two to a CU / 256 x 256):
    // 4: 7.1 / 13.9 / 20 / 25 / 47; 64: 12.9 / 13.9 / 20 / 26 / 50; 128: 22 / 13.8 / 20 / 26 / 51; 512: 75 / 16.6 / 21.1 / 26 / 50; 1024: 151 / 31 / 26.0 / 29 / 51;
    // 2048: 281 / 70 / 50 / 40 / 58; 8192 x 8192: 2239 / 439 / - / 317 / 256. Direct takes 3.5 us and 0.42 ns for each round of workgroups, k and 16 rows or columns of one
    // (64 x 16384 x 1024: 12.9 us, 64 x 512 x 8192: 20.0); 64 x 64 as much and 2.5 ns for each round and k (7.5 and 20.2). The largest two by their rounds, 40 and 64 us each.
    // Rows that begin at words take 0.37 and 5.2 ns (197 x 2049 x 1004: 7.9 / 8.8 us), others in arrays that do 0.65 and 6.9 (64 x 4097 x 4095: 27 / 30; 4 x 4099 x 4097: 10.1 /
    // 30), the rest 1.35 and 6.9.
    // Large ones at other addresses, whose bytes wait in registers: 5923 x 4002 x 1206 100 / 65 / 117 / 80, 1134 x 15690 x 3927 251 / 161 / 278 / 217 (64 x 64 / 128 x 128 one to a CU / two / 256 x 256).
    const int64_t tiles64 = ceil_div(p.M, (int64_t)64) * ceil_div(p.N, (int64_t)64), tiles128 = ceil_div(p.M, (int64_t)128) * ceil_div(p.N, (int64_t)128);
    const int64_t tiles256 = ceil_div(p.M, (int64_t)256) * ceil_div(p.N, (int64_t)256);
    int mt = 1;   // rows / 16 of a workgroup, direct
    auto direct_cost = [&](int rows16) { return ceil_div(ceil_div(p.M, (int64_t)(16 * rows16)) * ceil_div(p.N, (int64_t)16), (int64_t)256) * (rows16 + 1); };
    for (int rows16 = 2; rows16 <= 4; rows16 *= 2)
        if (direct_cost(rows16) < direct_cost(mt)) mt = rows16;
    const int per_tile = aligned ? 6 : !words ? 5 : p.K % 4 ? 10 : 15;
    const int form = tuning().qlin_form;
    const int pick = form >= 0 ? form : direct_cost(mt) <= per_tile * ceil_div(tiles64, (int64_t)512) ? 0 : tiles64 <= 512 ? 1 : tiles128 <= 256 || !aligned ? 2 : 40 * ceil_div(tiles128, (int64_t)512) <= 64 * ceil_div(tiles256, (int64_t)256) ? 3 : 4;
    if (pick == 4) tile(Int<2>{}, Int<4>{}, Int<4>{}, Int<2>{}, Int<2>{}, Int<128>{}, 1);
    else if (pick == 3) tile(Int<2>{}, Int<2>{}, Int<2>{}, Int<2>{}, Int<2>{}, Int<128>{}, 2);
    else if (pick == 2) tile(Int<2>{}, Int<4>{}, Int<2>{}, Int<1>{}, Int<3>{}, Int<128>{}, 1);
    else if (pick == 1) tile(Int<2>{}, Int<2>{}, Int<1>{}, Int<1>{}, Int<2>{}, Int<256>{}, 2);
    else if (mt == 1) direct(Int<1>{});
    else if (mt == 2) direct(Int<2>{});
    else direct(Int<4>{});
    return fits;
}

}  // namespace mi355x

extern "C" int mi355x_quantized_linear(const int8_t* X, const int8_t* W, const float* x_scale, const float* w_scale, const void* bias, const void* residual,
                                       void* Y, int64_t M, int64_t N, int64_t K, int64_t x_scale_count, int64_t w_scale_count, int activation, int type,
                                       void* stream) {
    using namespace mi355x;
    MI355X_REQUIRE(M >= 0 && N >= 0 && K >= 0, "quantized_linear: negative extent (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
    MI355X_REQUIRE(is_mixed_type(type), "quantized_linear: element type %d", type);
    MI355X_REQUIRE(activation >= MI355X_ACT_NONE && activation <= MI355X_ACT_SILU, "quantized_linear: activation %d", activation);
    MI355X_REQUIRE(K < (int64_t)1 << 17, "quantized_linear: K=%lld: sums of 2^17 products and more do not fit 32 bits", (long long)K);
    MI355X_REQUIRE(x_scale_count == 1 || x_scale_count == M, "quantized_linear: x_scale holds %lld values, expected 1 or M=%lld", (long long)x_scale_count, (long long)M);
    MI355X_REQUIRE(w_scale_count == 1 || w_scale_count == N, "quantized_linear: w_scale holds %lld values, expected 1 or N=%lld", (long long)w_scale_count, (long long)N);
    if (M == 0 || N == 0) return MI355X_OK;
    MI355X_REQUIRE((K == 0 || (X && W)) && x_scale && w_scale && Y, "quantized_linear: null pointer");
    MI355X_REQUIRE(M < (int64_t)1 << 31 && N < (int64_t)1 << 31, "quantized_linear: too large");
    QLinArgs p = {X, W, x_scale, w_scale, bias, residual, Y, M, N, K, x_scale_count != 1, w_scale_count != 1, activation, 0, 0};
    bool fits = true;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        hipStream_t st = static_cast<hipStream_t>(stream);
        if (activation == MI355X_ACT_RELU) fits = launch_qlin<T, MI355X_ACT_RELU>(p, st);
        else if (activation == MI355X_ACT_GELU) fits = launch_qlin<T, MI355X_ACT_GELU>(p, st);
        else if (activation == MI355X_ACT_SILU) fits = launch_qlin<T, MI355X_ACT_SILU>(p, st);
        else fits = launch_qlin<T, MI355X_ACT_NONE>(p, st);
    });
    MI355X_REQUIRE(fits, "quantized_linear: too large");
    return check_launch("quantized_linear");
}
