// A square tile of a product of 16-bit numbers on the matrix cores, with float32 sums: the loop that the products of
// muon.hip and indexed.hip share.
//
// Four wavefronts share a tile of BT x BT, a quarter each.  Its operands come in chunks from memory straight to LDS, 16
// bytes a lane, several chunks ahead.  An operand whose rows run along the sum ("by rows") lies in LDS as rows of 64
// numbers; one whose rows are the sum index ("by sums", TR) as it is in memory, and is read with the transposing LDS load.
// Within a row of LDS the 16-byte pieces are permuted (by the lanes' source addresses: LDS itself is filled in lane order)
// so that the reads, 16 bytes of 16 rows or 32 or 64 bytes of 4 rows, meet every bank once.
//
// Operands are read from LDS between the products of the 32 numbers before, which also cover the loads of chunks to come.
// One barrier a chunk, before its last products: by then everyone has read all of it (its place is free) and the next
// chunk has arrived.
//
// A chunk of 64 numbers takes 1.95 us with tiles of 256 (1.1 PFLOP/s on 256 CUs; a large library product reaches 1.47
// here), 1.1 with 192, 1.05 with two of 128 a CU, 0.23 with 64.
#pragma once

#include <type_traits>

#include "common.h"

namespace mnx {
namespace tile16 {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 brain8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kRow = 64;  // numbers of a row's chunk: 64 k, or 32 k of pairs (16 hi, then their 16 lo)

// Chunks in LDS at a time: as many as leave one workgroup (two of 128) a CU.
constexpr int stages(int tile) { return tile == 256 ? 2 : tile == 192 ? 3 : tile == 128 ? 2 : 6; }
constexpr int lds_numbers(int tile) { return 2 * stages(tile) * tile * kRow; }

template <bool BF16>
__device__ __forceinline__ f32x16 mfma(const short8v& a, const short8v& b, const f32x16& c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(brain8, a), __builtin_bit_cast(brain8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// 16 bytes a lane to LDS, lane by lane from `to` on (M0); from base + offset (bytes), or from an address a lane.  In
// assembly, because for the builtin the compiler waits for every such load before the next read of LDS, also of other
// memory there.  The caller waits (vmcnt) and has a barrier before anyone reads what has come, and before it ends.
//
// A load must not begin within five wait states of a vector instruction's write of its scalar base (a lane that was read,
// say), and the compiler does not look into the statement: the base passes through a scalar move, which waits by itself, and
// is the state that M0 needs, too.
__device__ __forceinline__ void load_lds(const void* base, uint32_t offset, void* to) {
    const uint32_t m0 = uint32_t(uintptr_t((__attribute__((address_space(3))) char*)to));
    const void* from;
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0"
                 : "=&s"(from)
                 : "s"(m0), "v"(offset), "s"(base)
                 : "memory", "m0");
}
__device__ __forceinline__ void load_lds(const void* from, void* to) {
    const uint32_t m0 = uint32_t(uintptr_t((__attribute__((address_space(3))) char*)to));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(m0), "v"(from) : "memory", "m0");
}

// The transposing read: of 16 lanes, four read 16 columns of one row, and lane l gets column l's four rows.  From `lo` and
// `hi`, four rows on: eight rows of a column.
__device__ __forceinline__ short8v read_tr(const void* lo, const void* hi) {
    typedef __attribute__((address_space(3))) short4v* P;
    const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)lo), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)hi);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// LDS that one lane wrote is read by others of the wavefront.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Tile `u` of a launch of up(units, 128) workgroups: 16 tiles next to each other run on one XCD (workgroups are dealt to
// the eight in turn).
__device__ __forceinline__ uint32_t unit_of_block() {
    return (((blockIdx.x >> 7) << 3 | (blockIdx.x & 7)) << 4) | (blockIdx.x >> 3 & 15);
}

// By rows: the n-th load of a chunk brings row `row + 32 n`, and of it the 16 bytes at number `number` of the chunk.
struct RowPlace {
    int row, number;
};
__device__ __forceinline__ RowPlace row_place() {
    const int lane = threadIdx.x & 63, row = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 8 + (lane >> 3);
    return {row, ((lane & 7) ^ ((row >> 1) & 7)) << 3};  // 32 rows on, pieces turn alike
}

// Of a piece in the row of sum k: pairs' hi and lo, 32 bytes each of two groups, or 64 bytes of a row.
template <int BT, int PL>
__device__ __forceinline__ int turn_of(int k) {
    return PL == 2 ? (k & 1) << 1 | (k & 2) << 2 : BT % 128 ? ((k >> 1) & 1) << 2 : (k & 3) << 2;
}
// By sums: the n-th load of a chunk brings, of sum `sum`, the 16 bytes at number `number` of the tile's columns.
struct SumPlace {
    int sum, number;
};
template <int BT, int PL>
__device__ __forceinline__ SumPlace sum_place(int n) {
    constexpr int PIECES = PL * BT / 8;
    const int piece = (n * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 64 + int(threadIdx.x & 63);
    const int k = piece / PIECES;
    return {k, (piece % PIECES ^ turn_of<BT, PL>(k)) << 3};
}

// acc[m][n][q] is of row 32 m + l32 and column 32 n + 8 (q / 4) + 4 half + q % 4 of the wavefront's part, which begins at
// row BT / 2 (wave % 2) and column BT / 2 (wave / 2); l32 and half are the lane's.
template <int BT>
using Acc = f32x16[BT / 64][BT / 64];

template <int BT>
__device__ __forceinline__ void clear(Acc<BT>& acc) {
#pragma unroll
    for (int m = 0; m < BT / 64; ++m)
#pragma unroll
        for (int n = 0; n < BT / 64; ++n)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[m][n][q] = 0.f;
}

// acc += the sum over `chunks` (1 or more) chunks of I's rows times J's columns.  load(c, n, to), n from 0 to 2 FETCH - 1
// (FETCH = BT / 32), issues the n-th load of chunk c into `to`: of I first, then of J; ahead(c) is called some time before
// chunk c's first.  PL = 2: I and J are of pairs.  When it ends, every load has come, but others may still read LDS.
template <int BT, int PL, bool TRI, bool TRJ, bool BF16, typename Load, typename Ahead>
__device__ __forceinline__ void products(short* lds, int chunks, Acc<BT>& acc, Load load, Ahead ahead) {
    constexpr int W = BT / 2, MT = W / 32, STAGES = stages(BT), SIDE = BT * kRow, FETCH = BT / 32;
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave & 1, wj = wave >> 1;
    auto fetch = [&](int c, int n, int stage) { load(c, n, lds + stage * 2 * SIDE + (n * 4 + wave) * 512); };
    // operands of 32 numbers: k 0 to 15 and 16 to 31, or hi and lo
    struct Frags {
        short8v i[2][MT], j[2][MT];
    };
    const int trow = 8 * half + ((lane & 15) >> 2), turn = (l32 >> 1) & 7;
    auto read = [&](auto tr, int part, int sub, int h, int m, const short* b) {
        if constexpr (!decltype(tr)::value) {
            return *reinterpret_cast<const short8v*>(b + (part * W + m * 32 + l32) * kRow + (((4 * sub + 2 * h + half) ^ turn) << 3));
        } else {  // four sums on turn alike
            const int k = trow + 32 / PL * sub + (PL == 1 ? 16 * h : 0), col = part * W + m * 32 + (l32 & 16);
            const int in = PL == 1 ? col + (lane & 3) * 4 : 2 * col + 16 * h + (lane & 3) * 4;
            const short* q = b + k * (PL * BT) + (((in >> 3) ^ turn_of<BT, PL>(trow)) << 3) + (in & 4);
            return read_tr(q, q + 4 * PL * BT);
        }
    };
    const std::integral_constant<bool, TRI> tri;
    const std::integral_constant<bool, TRJ> trj;
    auto read_both = [&](Frags& f, int h, int m, int stage, int sub) {
        const short* b = lds + stage * 2 * SIDE;
        f.j[h][m] = read(trj, wj, sub, h, m, b + SIDE);
        f.i[h][m] = read(tri, wi, sub, h, m, b);
    };
    // The products of `now`, with the reads of `next` (32 numbers of a chunk) and `loads` between them.
    auto multiply = [&](const Frags& now, Frags& next, int stage, int sub, auto loads) {
        // k by k, or of pairs lo hi, hi lo, hi hi
        constexpr int GROUPS = PL == 1 ? 2 : 3, HI[3] = {0, 1, 0}, HJ[3] = {PL == 1 ? 0 : 1, PL == 1 ? 1 : 0, 0};
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if (g < 2) read_both(next, g, m, stage, sub);
                loads(g * MT + m);
#pragma unroll
                for (int n = 0; n < MT; ++n) acc[m][n] = mfma<BF16>(now.j[HJ[g]][n], now.i[HI[g]][m], acc[m][n]);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    const auto nothing = [](int) {};
    // a chunk's loads, shared out over the first 2 MT products
    auto loads_of = [&](int c, int stage) {
        return [=, &fetch](int at) {
            constexpr int PER = (2 * FETCH + 2 * MT - 1) / (2 * MT);
#pragma unroll
            for (int n = at * PER; n < (at + 1) * PER; ++n)
                if (n < 2 * FETCH) fetch(c, n, stage);
        };
    };
    auto barrier = [] {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto next_of = [](int stage) { return stage + 1 == STAGES ? 0 : stage + 1; };
    Frags f0, f1;
    int stage = 0, c = 0;
#pragma unroll 1
    for (int k = 0; k < min(STAGES, chunks); ++k) {
        ahead(k);
#pragma unroll
        for (int n = 0; n < 2 * FETCH; ++n) fetch(k, n, k);
    }
    ahead(min(STAGES, chunks - 1));
    if (chunks >= STAGES) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * FETCH * (STAGES - 1)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    barrier();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < MT; ++m) read_both(f0, h, m, 0, 0);
    // The last products of chunk c, whose operands are in `now`, and the first operands of the next.  MORE: chunk
    // c + STAGES goes where c was.
    auto last_of = [&](const Frags& now, Frags& next, auto more) {
        // (STAGES - 2) chunks behind the next may still be out
        if constexpr (decltype(more)::value)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(2 * FETCH * (STAGES - 2)) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        barrier();
        const int free = stage;
        stage = next_of(stage);
        if constexpr (decltype(more)::value) multiply(now, next, stage, 0, loads_of(c + STAGES, free));
        else multiply(now, next, stage, 0, nothing);  // after the last chunk it reads what nobody uses
        ++c;
    };
    const std::true_type more;
    const std::false_type rest;
    multiply(f0, f1, stage, 1, nothing);
#pragma unroll 1
    while (c + STAGES < chunks) {
        last_of(f1, f0, more);
        multiply(f0, f1, stage, 1, nothing);
        ahead(min(c + STAGES, chunks - 1));
    }
#pragma unroll 1
    while (c + 1 < chunks) {
        last_of(f1, f0, rest);
        multiply(f0, f1, stage, 1, nothing);
    }
    last_of(f1, f0, rest);
}

}  // namespace tile16
}  // namespace mnx
