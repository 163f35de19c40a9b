// Matrix product of the vocabulary losses (gfx950): C[m][n] = sum_k X(m, k) Y(n, k), bfloat16
// operands, float32 sums, for the three products of a vocabulary head:
//
//   logits   Z = H W^T      X = H [m][k], Y = W [n][k]      both rows run along the contraction
//   dhidden  G W            X = G [m][k], Y = W [k][n]      Y's rows run along the output
//   dweight  G^T H          X = G [k][m], Y = H [k][n]      both rows run along the outputs
//
// so no operand is ever transposed in memory: an operand whose rows run along the output is
// staged as it lies and read with the LDS transpose read.
//
// One workgroup of 8 waves makes a BM x BN tile in steps of 64 along the contraction.  A step's
// operands go from memory to LDS by LDS DMA (1 KB an instruction, no registers) into one of NST
// stages; a wave reads the fragments of one half step (32) while its matrix instructions work on
// the other half, so a step has one barrier, and a stage is refilled as soon as the second
// half's fragments have left it, a whole step before it is read again.
//
// The matrix instruction is given Y as its row operand and X as its column operand: the
// accumulator then holds four consecutive n of one m in each lane, which is what row-major
// outputs store at once and what a softmax over n reduces inside a lane.
//
// LDS layouts (16-byte chunks, swizzled by row so that fragment reads spread over the banks):
//   rows along k  ("RowK"): [BM][64], 128-byte rows, chunk c of row r at c ^ (r & 7), read 16
//                 bytes at a time; where the other operand needs transpose reads, chunk c at
//                 c ^ ((r >> 1) & 7) and read 8 + 8 bytes in the transpose read's order of k
//                 (slots 0-3 = k0 + 4q + e, 4-7 = k0 + 16 + 4q + e).
//   rows along the output ("RowN"): [64][BN], chunk c of row r at c ^ (2 (r & 7)), read by
//                 ds_read_b64_tr_b16.
//
// 8192 x 65536 x 5120: 4.0-4.2 ms in the three layouts (1.32-1.38 PFLOP/s), the card at its power limit
// (1.85 GHz; the matrix cores busy 65 % of the time, no bank conflicts, 81 % L2 hits).  64 tokens'
// logits read a weight of 0.34 GB in 61 us (5.5 TB/s).
#pragma once

#include <type_traits>

#include "wkv7_io.h"

namespace vocab {

using wkv7::f32x4_t;

constexpr int BK = 64;  // contraction per step

enum Lay { RowK, RowN };

// One operand: rows of `ld` elements.  RowK: outer index -> row, `outer` valid rows, the
// contraction's `K` elements in every row.  RowN: contraction index -> row, `inner` valid rows,
// `outer` elements valid in a row (a multiple of 8).  Rows and columns beyond are read from the
// last valid place; the other operand is zero there, or the output is not stored.  RowN with
// `twice`: one step of rows 0 .. 31 and again 0 .. 31.
struct Operand {
    const uint16_t* p;
    long ld;
    int outer, inner;
    bool twice = false;
};

struct Tiles {
    int m, n;     // tiles of the output
    int splits;   // parts of the contraction
    int steps;    // steps of one part (the last may have fewer)
    int all;      // steps in all
    int group;    // m tiles that run together
    int total;    // tiles in all: m n splits
};

struct Where {
    int m, n, part;
};
// Workgroup b % (the grid, where that is smaller, a multiple of 8) runs on XCD b % 8: each XCD takes a run of consecutive tiles, ordered in groups of
// `group` m tiles that share the n tiles they walk over, so that an XCD's L2 serves both operands.
__device__ __forceinline__ Where tile_of(const Tiles& t, int b) {
    const int each = t.total >> 3;
    int id = b < each * 8 ? (b & 7) * each + (b >> 3) : b;
    const int mn = t.m * t.n;
    Where w;
    w.part = id / mn;
    id -= w.part * mn;
    const int per = t.group * t.n, g = id / per, first = g * t.group;
    const int size = min(t.m - first, t.group);
    id -= g * per;
    w.n = id / size;
    w.m = first + (id - w.n * size);
    return w;
}

// LDS DMA of 1 KB into `lds` (byte address), from base + voff.
__device__ __forceinline__ void dma(uint32_t lds, const uint8_t* base, uint32_t voff) {
    wkv7::dma_kb(lds, wkv7::dma_rsrc(base, 0xffffffffu), voff, 0);
}

// The stage loader of one operand for a wave: its 1 KB pieces w, w + 8, ... of a [B][64] or
// [64][B] tile.
template <Lay L, int B, bool PERM> struct Loader {
    static constexpr int PIECES = B * BK * 2 / 1024 / 8;   // per wave
    static constexpr int PER = L == RowK ? 8 : 512 / B;    // rows in a piece
    static_assert(B * BK * 2 % 8192 == 0 && (L == RowK || B == 256 || B == 128 || B == 64), "tile");
    const uint8_t* base;
    uint32_t row, col, ld2;
    uint32_t mask;  // of a row's number (RowN)
    uint32_t limit; // RowK: offset of the tile's last valid row
    int rows_left;  // RowN: valid rows from the step's first

    __device__ __forceinline__ Loader(const Operand& o, int x0, int k0, int wave, int lane) {
        ld2 = (uint32_t)(o.ld * 2);
        if constexpr (L == RowK) {
            const int r = 8 * wave + (lane >> 3);
            const int c = (lane & 7) ^ (PERM ? (r >> 1) & 7 : r & 7);
            base = reinterpret_cast<const uint8_t*>(o.p + (long)x0 * o.ld + k0);
            mask = ~0u;
            row = r * ld2;
            col = 16 * c;
            limit = (uint32_t)max(min(o.outer - x0, B) - 1, 0) * ld2;  // (of the tile: 32 bits hold its rows' offsets)
            rows_left = 0;
        } else {
            constexpr int CH = B / 8;  // chunks in a row
            const int r = PER * wave + lane / CH;
            const int c = (lane & (CH - 1)) ^ ((2 * (r & 7)) & (CH - 1));
            base = reinterpret_cast<const uint8_t*>(o.p + (long)k0 * o.ld + x0);
            mask = o.twice ? 31u : ~0u;
            row = (r & mask) * ld2;
            col = 2 * min(8 * c, o.outer - x0 - 8);
            rows_left = o.inner - k0;
            limit = 0;
        }
    }
    // piece j of the next step into the tile at `lds`; advance() after the last one
    __device__ __forceinline__ void issue(uint32_t lds, int j, int wave) const {
        const uint32_t last = L == RowK ? limit : (uint32_t)max(min(rows_left, BK) - 1, 0) * ld2;
        const uint32_t r = min(row + ((uint32_t)(8 * PER * j) & mask) * ld2, last);
        dma(lds + (uint32_t)(wave + 8 * j) * 1024, base, r + col);
    }
    // to the next step (behind a workgroup's last one the loader stays: its pieces are then not used)
    __device__ __forceinline__ void advance(bool more) {
        if constexpr (L == RowK) base += more ? BK * 2 : 0;
        else {
            base += more ? (long)BK * ld2 : 0;
            rows_left -= more ? BK : 0;
        }
    }
    // or to another tile's first step
    __device__ __forceinline__ void move(bool more, bool jump, const Loader& to) {
        advance(more);
        base = jump ? to.base : base;
        if constexpr (L == RowK) {
            limit = jump ? to.limit : limit;
        } else {
            rows_left = jump ? to.rows_left : rows_left;
            col = jump ? to.col : col;
        }
    }
};

// The fragment reader of one operand for a wave: fragment i = outer 16 i .. + 15 from the wave's
// first, half step h, from the tile at LDS byte address `at`.
template <Lay L, int B, bool PERM> struct Reader {
    uint32_t a;
    __device__ __forceinline__ Reader(int x0, int lane) {
        const int r16 = lane & 15, q = lane >> 4;
        if constexpr (L == RowK) {
            const int r = x0 + r16;
            if constexpr (PERM) a = r * 128 + 8 * (q & 1) + 16 * ((q >> 1) ^ ((r >> 1) & 7));
            else a = r * 128 + 16 * (q ^ (r & 7));
        } else {
            constexpr int CH = B / 8;
            const int r = 4 * q + (r16 >> 2);
            const int c = (x0 / 8 + ((r16 & 3) >> 1)) ^ ((2 * (r & 7)) & (CH - 1));
            a = r * (B * 2) + 16 * c + 8 * (r16 & 1);
        }
    }
    __device__ __forceinline__ uint4 get(const uint8_t* lds, uint32_t at, int i, int h) const {
        if constexpr (L == RowK) {
            if constexpr (PERM) {
                const uint8_t* p = lds + at + 2048 * i;
                const uint2 lo = *reinterpret_cast<const uint2*>(p + (a ^ (64 * h)));
                const uint2 hi = *reinterpret_cast<const uint2*>(p + (a ^ (64 * h + 32)));
                return make_uint4(lo.x, lo.y, hi.x, hi.y);
            } else {
                return *reinterpret_cast<const uint4*>(lds + at + 2048 * i + (a ^ (64 * h)));
            }
        } else {
            // (outer 16 i is chunk 2 i: an exclusive or inside the wave's first chunks, which are a multiple of its fragments)
            const uint8_t* p = lds + at + (a ^ (32 * i)) + 32 * h * (B * 2);
            const uint2 lo = wkv7::tr_at(reinterpret_cast<const uint16_t*>(p));
            const uint2 hi = wkv7::tr_at(reinterpret_cast<const uint16_t*>(p + 16 * (B * 2)));
            return make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
    }
};

// this wave's LDS reads done and all but its last N DMAs, then everyone's (by the builtins: the
// compiler counts the reads that are still out, and knows here that none is)
template <int N> __device__ __forceinline__ void wait_barrier() {
    wkv7::vm_wait_n<N>();
    __builtin_amdgcn_s_waitcnt(0xc07f);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// threadIdx.x where a tile is finished: what follows from it is made there again, not held in registers
// through the multiplication
__device__ __forceinline__ int thread_here() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

struct Place {
    int m0, n0, step0, steps;
};

// BM x BN tiles: WM x WN waves of TM x TN fragments, NST stages.  go() makes a workgroup's tiles one
// after the other: next(place) says which (false: no more), done(place) is called with each tile's
// acc[tn][tm] (lane: n = 16 tn + 4 (lane / 16) + e, m = 16 tm + lane % 16 from the wave's first).
// While a tile's last steps are multiplied and done() works in LDS of its own (epilogue()), the
// next tile's first stages are on their way (a workgroup's tiles have more than NST steps, or it has one;
// one tile a workgroup throughout: 2604 tokens' logits of 53714 at D = 768 336 us for 295, 365 tokens'
// dweight of 60000 x 2560 159 for 144, with 80 steps and more, at the power limit, the same).  Shapes whose
// stages leave no LDS for that (KEPT false) make one tile, and done() writes where the stages were.
template <int BM_, int BN_, int WM_, int WN_, int NST_, Lay LX_, Lay LY_> struct Product {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NST = NST_;
    static constexpr Lay LX = LX_, LY = LY_;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    static constexpr bool PERM = LX == RowN || LY == RowN;
    static constexpr int STAGE = (BM + BN) * BK * 2;
    static constexpr int EPILOGUE = TN * 4096 > 9216 ? TN * 4096 : 9216;
    static constexpr bool KEPT = NST * STAGE + EPILOGUE <= 163840;
    static constexpr int LDS = NST * STAGE + (KEPT ? EPILOGUE : 0);
    static constexpr int THREADS = 512;
    static_assert(WM * WN == 8, "eight waves");
    using LoadX = Loader<LX, BM, PERM>;
    using LoadY = Loader<LY, BN, PERM>;
    static constexpr int PIECES = LoadX::PIECES + LoadY::PIECES;

    __device__ static __forceinline__ uint8_t* epilogue(uint8_t* lds) { return lds + (KEPT ? NST * STAGE : 0); }

    f32x4_t acc[TN][TM];

    // SHORT, for tiles of few steps: what is loaded ahead lies any number of tiles ahead; else no further
    // than in the next tile.  (33 tokens' dweight of 56136 x 5120, one step a tile: 142 us with one tile a
    // workgroup, 113 so, 5.1 TB/s)
    template <bool SHORT, class Next, class Done>
    __device__ __forceinline__ void go(uint8_t* lds, const Operand& X, const Operand& Y, Place at, Next next, Done done) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
        LoadX lx(X, at.m0, at.step0 * BK, wave, lane);
        LoadY ly(Y, at.n0, at.step0 * BK, wave, lane);
        const Reader<LX, BM, PERM> rx((wave / WN) * TM * 16, lane);
        const Reader<LY, BN, PERM> ry((wave % WN) * TN * 16, lane);
        Place far = at;  // (SHORT: where the loaders are)
        Next beyond = next;
        int step = 0;
        auto forward = [&] {
            if (step + 1 < far.steps) {
                step++;
                lx.advance(true);
                ly.advance(true);
            } else if (Place to; beyond(to)) {
                far = to, step = 0;
                lx = LoadX(X, to.m0, to.step0 * BK, wave, lane);
                ly = LoadY(Y, to.n0, to.step0 * BK, wave, lane);
            }
        };
        auto piece = [&](int stage, int j) {
            if (j < LoadX::PIECES) lx.issue(lds0 + stage * STAGE, j, wave);
            else ly.issue(lds0 + stage * STAGE + BM * BK * 2, j - LoadX::PIECES, wave);
        };
#pragma unroll
        for (int s = 0; s < NST; s++) {
#pragma unroll
            for (int j = 0; j < PIECES; j++) piece(s, j);
            if constexpr (SHORT) {
                forward();
            } else {
                lx.advance(s + 1 < at.steps);
                ly.advance(s + 1 < at.steps);
            }
        }
        wait_barrier<(NST - 1) * PIECES>();

        // One half step is TN groups of TM matrix instructions.  A y fragment's registers take the
        // next half's fragment as soon as its group is done; x, used by every group, has two sets.
        uint4 x0[TM], x1[TM], y[TN];
        auto read_x = [&](uint4 (&x)[TM], int stage, int i, int h) { x[i] = rx.get(lds, stage * STAGE, i, h); };
        auto read_y = [&](int stage, int i, int h) { y[i] = ry.get(lds, stage * STAGE + BM * BK * 2, i, h); };
        auto group = [&](const uint4 (&x)[TM], int tn) {
#pragma unroll
            for (int tm = 0; tm < TM; tm++) acc[tn][tm] = wkv7::mma32(acc[tn][tm], y[tn], x[tm]);
        };
        // groups G0 .. TN - 1; behind each, what there is of a stage's refill and of the next half's
        // fragments: y as its registers come free, x spread over the groups
        auto groups = [&](const uint4 (&x)[TM], uint4 (&xn)[TM], int stage, int h, auto first, auto fill, int fstage) {
            constexpr int G0 = decltype(first)::value, NG = TN - G0;
#pragma unroll
            for (int g = G0; g < TN; g++) {
                group(x, g);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (decltype(fill)::value) {
#pragma unroll
                    for (int j = 0; j < PIECES; j++)
                        if (G0 + j * NG / PIECES == g) piece(fstage, j);
                }
#pragma unroll
                for (int i = 0; i < TM; i++)
                    if (G0 + i * (NG - 1) / TM == g) read_x(xn, stage, i, h);
#pragma unroll
                for (int i = 0; i < TN; i++)
                    if ((i > G0 ? i : G0) == g) read_y(stage, i, h);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        constexpr int BG = TN < 8 || PERM ? 0 : 3;  // groups of the second half ahead of the barrier
        using None = std::integral_constant<int, 0>;
        using Late = std::integral_constant<int, BG>;
        int cur = 0;
        for (;;) {
            Place to;
            const bool more = KEPT && next(to);
            if (!more) to = at;
            const LoadX tx(X, to.m0, to.step0 * BK, wave, lane);
            const LoadY ty(Y, to.n0, to.step0 * BK, wave, lane);
#pragma unroll
            for (int tn = 0; tn < TN; tn++)
#pragma unroll
                for (int tm = 0; tm < TM; tm++) acc[tn][tm] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < TM; i++) read_x(x0, cur, i, 0);
#pragma unroll
            for (int i = 0; i < TN; i++) read_y(cur, i, 0);
            __builtin_amdgcn_s_waitcnt(0xc07f);  // (so that what is out at the loop's start is what its end left)
            auto multiply = [&](auto move) {
                groups(x0, x1, cur, 1, None{}, std::false_type{}, 0);
                // (the stage's last reads complete under these)
#pragma unroll
                for (int g = 0; g < BG; g++) group(x1, g);
                __builtin_amdgcn_sched_barrier(0);
                // the next stage has landed, and every wave has read all of this one
                wait_barrier<(NST - 2) * PIECES>();
                const int then = cur + 1 == NST ? 0 : cur + 1;
                groups(x1, x0, then, 0, Late{}, std::true_type{}, cur);
                move();
                cur = then;
            };
            // step s loads step s + NST; the last ones, which load the next tile's, in a loop of their own
            // (the choice in the long one costs 2 %)
            if constexpr (SHORT) {
                for (int s = 0; s < at.steps; s++) multiply(forward);
            } else {
                int s = 0;
                for (; s < at.steps - NST - 1; s++)
                    multiply([&] {
                        lx.advance(true);
                        ly.advance(true);
                    });
                for (; s < at.steps; s++)
                    multiply([&] {
                        const int left = at.steps - NST - 1 - s;
                        lx.move(more && left < 0, more && left == 0, tx);
                        ly.move(more && left < 0, more && left == 0, ty);
                    });
            }
            if constexpr (!KEPT) {
                wkv7::vm_wait_n<0>();
                __syncthreads();
            }
            done(at);
            if (!more) break;
            at = to;
        }
        wkv7::vm_wait_n<0>();  // (before the workgroup's LDS is another's)
    }
};

// The workgroup's tile of 16-bit values to memory, whole rows at a time: an accumulator lane holds
// 8 bytes of a row, which stored as they are reach memory as 32-byte pieces of 16 rows (8192 x
// 65536 exponentials at D = 640: 1080 us, and 920 by whole rows; a weight gradient of 65536 x
// 5120 from 64 tokens 233 and 158).  Each wave turns its own tile, 16 rows at a time, in its own part of
// the epilogue's LDS (16-byte chunk c of row r at c ^ (r mod chunks)).  pack(tn, tm): the lane's four
// values; put(m, n, v): eight values of row m from column n, both from the workgroup's first.
template <class P, class Pack, class Put> __device__ __forceinline__ void store_rows(uint8_t* lds, Pack pack, Put put) {
    constexpr int CH = P::TN * 2, ROW = CH * 16;  // chunks and bytes of a row of the wave's tile
    constexpr int EACH = CH < 4 ? 2 : 1;          // fragments of 16 rows at a time: 64 chunks or more
    static_assert(P::TM % EACH == 0 && 8 * EACH * 16 * ROW <= P::EPILOGUE, "tile");
    const int thread = thread_here(), lane = thread & 63, wave = thread >> 6, r16 = lane & 15, q = lane >> 4;
    uint8_t* mine = P::epilogue(lds) + wave * (EACH * 16 * ROW);
    const int c = lane & (CH - 1), m0 = (wave / P::WN) * P::TM * 16, n = (wave % P::WN) * P::TN * 16 + 8 * c;
#pragma unroll
    for (int t0 = 0; t0 < P::TM; t0 += EACH) {
#pragma unroll
        for (int t = 0; t < EACH; t++)
#pragma unroll
            for (int tn = 0; tn < P::TN; tn++)
                *reinterpret_cast<uint2*>(mine + (16 * t + r16) * ROW + (((2 * tn + (q >> 1)) ^ (r16 & (CH - 1))) << 4) + 8 * (q & 1)) = pack(tn, t0 + t);
        wkv7::wave_lds_fence();
#pragma unroll
        for (int i = 0; i < EACH * 16 * CH / 64; i++) {
            const int r = i * (64 / CH) + lane / CH;
            put(m0 + 16 * t0 + r, n, *reinterpret_cast<const uint4*>(mine + r * ROW + ((c ^ (r & (CH - 1))) << 4)));
        }
        wkv7::wave_lds_fence();
    }
}

}  // namespace vocab
