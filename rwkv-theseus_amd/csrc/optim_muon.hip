// Orthogonalised updates (C ABI: include/theseus_muon.h), gfx950.
//
// X_0 = s u / max(|u|_F, eps) and, `steps` times with p the short side,
//
//   A = X X^T (X^T X where X is tall)      the lower triangle's tiles, each stored on both sides
//   B = s^2 a I + b A + (c / s^2) A^2      the same: A is symmetric, so A^2 = A A^T
//   X = (1 / s^2) B X (X B)
//
// p^2 q + p^3 + 2 p^2 q products and sums a step instead of 2 p^2 q + 2 p^3 + 2 p^2 q, on the matrix
// cores with vocab_gemm.h's tiles: a wide X is read along its rows for A and along its columns for
// B X, a tall one the other way round, so no matrix is ever transposed in memory.  The list's
// matrices share every launch: workgroups find their matrix in the kernel's arguments.
//
// Numerics.  Operands are float16: bfloat16 has 8 times their rounding, and the polynomial magnifies
// it (a Gaussian 768 x 768: 1.0e-2 from the exact result instead of 1.3e-3, where rounding the result
// to bfloat16 costs 1.7e-3).  s, a power of two up to 32 near sqrt(p), keeps their values (X near 1 / sqrt(q), A near 1
// after the first steps and s^2 / p before, B up to a s^2) inside float16's range.  Where u has few strong
// directions, rounding X would add to it a matrix outside of its row and column spaces, which the polynomials
// raise by a each step, 485 in five, while the strong directions stay at 1 (rank 64 of 768: 2.3e-2 off, rank 1:
// 0.15).  The other roundings' errors lie inside one of these spaces and grow as X does.  So X is held in two
// halves, hi + lo / 2048: hi goes into the products, a lo is added to the next X; only the last step's X, whose
// rounding is raised 3.4 times at most, is hi alone.  At most 2.6e-3 on all spectra that were tried.
//
// What bounds it (the ten matrices of a layer of width 5120, a step in 10.8 ms: Gram matrices 5 x 513 us, squares 5 x 536,
// updates 5 x 1003, momentum and X_0 497).  The products' cores run at 1.3 PFLOP/s, the card's power limit; a tile's end, in
// which all CUs write at once, is 9 % of a Gram matrix' time (of 433 us in tiles of 256), the last round, in
// quarters, 80 us of it.  Small matrices are bound by their launches, 4 to 8 us each, three a step.
#include "../../include/theseus_muon.h"
#include "../../include/theseus_wkv7.h"

#include <math.h>

#include <type_traits>

#include "optim_norm.h"
#include "vocab_gemm.h"

namespace muon {

using namespace vocab;
using wkv7::bf16_to_f32;
using wkv7::f32x2_to_bf16x2;

constexpr int MAX = 32;         // matrices of a launch
constexpr int TOGETHER = 1024;  // rows of a product whose tiles run together
constexpr int PIECE = 2048;     // elements of a workgroup of the passes ahead of the products, `each` times
constexpr int SPLITS = 8;       // of A's contraction at most
constexpr float LO = 2048.f;    // of X's second half, so that it is no subnormal

// One matrix.  Its part of the workspace: X hi, X lo, the next X hi and lo ([mp][np] each, zero
// beyond m and n), A and B ([pp][pp], pp the padded short side), and where A has few tiles SPLITS parts of it.
struct Matrix {
    const void* src;  // the gradient, or X
    long ld;          // of src
    float* momentum;  // null: orthogonalize
    void* dst;        // float32 param, or bfloat16 out
    uint16_t* ws;
    int m, n, mp, np;  // and padded to steps of the products
    int piece0, pieces, each;  // of the norm's partial sums; PIECEs of a workgroup
    float s;
    float keep, step;
    int fp32;  // src
    __device__ __host__ bool tall() const { return m > n; }
    __device__ __host__ int pp() const { return tall() ? np : mp; }
    __device__ long size() const { return (long)mp * np; }
    __device__ uint16_t* hi(int which) const { return ws + 2 * which * size(); }
    __device__ uint16_t* lo(int which) const { return hi(which) + size(); }
    __device__ uint16_t* gram() const { return ws + 4 * size(); }
    __device__ uint16_t* square() const { return gram() + (long)pp() * pp(); }
    __device__ float* parts() const { return reinterpret_cast<float*>(square() + (long)pp() * pp()); }  // of A, where it is split
};
struct List {
    int count;
    int first[MAX + 1];  // of each matrix' workgroups in this launch
    Matrix x[MAX];
};
static_assert(sizeof(List) < 4000, "kernel arguments");

// (all of them at once, a lane each: one wait instead of one a matrix)
__device__ __forceinline__ int which(const List& l, int b) {
    static_assert(MAX < 64, "lanes");
    const int lane = threadIdx.x & 63, n = l.count;
    if (n == 1) return 0;
    return __builtin_popcountll(__ballot(lane < n && l.first[min(lane, MAX)] <= b)) - 1;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint32_t half2_of(float x, float y) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, h2{(_Float16)x, (_Float16)y});
}
__device__ __forceinline__ float2 floats_of(uint32_t u) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 h = __builtin_bit_cast(h2, u);
    return make_float2((float)h[0], (float)h[1]);
}
// x, y -> hi; what that rounds away, times BY -> lo
template <int BY = (int)LO> __device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = half2_of(x, y);
    const float2 h = floats_of(hi);
    lo = half2_of((x - h.x) * BY, (y - h.y) * BY);
}

// ------------------------------------------------------------------------------ u, its norm, X_0
struct Update {
    float mu, nu;  // momentum, and 1 - momentum
    int nesterov;
    float factor;         // of the gradients, where result is null
    const float* result;  // of the norm pass: the factor, and whether nothing may change
    int skip;
    float eps;
};
__device__ __forceinline__ bool skipped(const Update& u) { return u.result && u.skip && u.result[2] != 0.f; }

template <typename T> struct Eight {
    typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));  // (rows may begin anywhere)
};
__device__ __forceinline__ void load8(float (&x)[8], const void* p, long at, int count, bool fp32) {
    if (count >= 8) {
        if (fp32) {
            const auto v = *reinterpret_cast<const Eight<float>::type*>(static_cast<const float*>(p) + at);
            for (int e = 0; e < 8; e++) x[e] = v[e];
        } else {
            const auto v = *reinterpret_cast<const Eight<uint16_t>::type*>(static_cast<const uint16_t*>(p) + at);
            for (int e = 0; e < 8; e++) x[e] = bf16_to_f32(v[e]);
        }
    } else {
        for (int e = 0; e < 8; e++)
            x[e] = e >= count ? 0.f : fp32 ? static_cast<const float*>(p)[at + e] : bf16_to_f32(static_cast<const uint16_t*>(p)[at + e]);
    }
}
__device__ __forceinline__ double block_sum(double x, double* red) {  // in every thread
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// momentum, and the sum of u^2 of a workgroup's rows: float32 values, float64 squares and sums (their squares may
// leave float32's range, and there are up to 2^34 of them)
__global__ __launch_bounds__(256) void momentum_norm(List l, Update u, double* __restrict__ sums) {
    __shared__ double red[4];
    if (skipped(u)) return;
    const int i = which(l, blockIdx.x), k = blockIdx.x - l.first[i];
    const Matrix& x = l.x[i];
    const float f = u.result ? u.result[1] : u.factor;
    const int per = (x.n + 7) / 8;
    const long all = (long)x.m * per;
    double sum = 0;
    for (int j = 0; j < x.each; j++) {
        const long c = ((long)k * x.each + j) * 256 + threadIdx.x;
        if (c >= all) break;
        const long row = c / per;
        const int col = (int)(c - row * per) * 8, count = x.n - col;
        float g[8];
        load8(g, x.src, row * x.ld + col, count, x.fp32);
        if (x.momentum) {
            float m[8];
            const long at = row * x.n + col;
            load8(m, x.momentum, at, count, true);
            for (int e = 0; e < 8; e++) {
                g[e] *= f;
                m[e] = u.mu * m[e] + u.nu * g[e];
            }
            if (count >= 8) {
                Eight<float>::type v;
                for (int e = 0; e < 8; e++) v[e] = m[e];
                *reinterpret_cast<Eight<float>::type*>(x.momentum + at) = v;
            } else {
                for (int e = 0; e < count; e++) x.momentum[at + e] = m[e];
            }
            for (int e = 0; e < 8; e++) g[e] = u.nesterov ? u.mu * m[e] + u.nu * g[e] : m[e];
        }
        for (int e = 0; e < 8; e++) sum += (double)g[e] * g[e];
    }
    sum = block_sum(sum, red);
    if (threadIdx.x == 0) sums[x.piece0 + k] = sum;
}

// X_0 in two halves, with zeros around it
__global__ __launch_bounds__(256) void scale_split(List l, Update u, const double* __restrict__ sums) {
    __shared__ double red[4];
    const int i = which(l, blockIdx.x), k = blockIdx.x - l.first[i];
    const Matrix& x = l.x[i];
    double sum = 0;
    for (int j = threadIdx.x; j < x.pieces; j += 256) sum += sums[x.piece0 + j];
    const double norm = sqrt(block_sum(sum, red));
    const float by = (float)(x.s / (norm < u.eps ? (double)u.eps : norm));  // (a NaN stays one)
    const float f = u.result ? u.result[1] : u.factor;
    const int per = x.np / 8;
    const long all = (long)x.mp * per;
    for (int j = 0; j < x.each; j++) {
        const long c = ((long)k * x.each + j) * 256 + threadIdx.x;
        if (c >= all) break;
        const long row = c / per;
        const int col = (int)(c - row * per) * 8, count = row < x.m ? x.n - col : 0;
        float g[8];
        load8(g, x.src, row * x.ld + col, count, x.fp32);
        if (x.momentum) {
            float m[8];
            load8(m, x.momentum, row * x.n + col, count, true);
            for (int e = 0; e < 8; e++) g[e] = u.nesterov ? u.mu * m[e] + u.nu * (g[e] * f) : m[e];
        }
        uint4 hi, lo;
        split(g[0] * by, g[1] * by, hi.x, lo.x);
        split(g[2] * by, g[3] * by, hi.y, lo.y);
        split(g[4] * by, g[5] * by, hi.z, lo.z);
        split(g[6] * by, g[7] * by, hi.w, lo.w);
        *reinterpret_cast<uint4*>(x.hi(0) + row * x.np + col) = hi;
        *reinterpret_cast<uint4*>(x.lo(0) + row * x.np + col) = lo;
    }
}

// ------------------------------------------------------------------------------ products
// A launch makes tiles from, from + 1, .. of the list, its workgroups one after the other: t-th of
// the launch -> its number, each XCD (t % 8) a run of consecutive ones, so that its L2 serves
// both operands.
struct Span {
    int from, count;
    bool quarters;   // of tiles of twice the side
    int splits = 1;  // parts of each tile's contraction, one after the other
};
__device__ __forceinline__ int number_of(const Span& s, int t) {
    const int each = s.count >> 3;
    return t < each * 8 ? (t & 7) * each + (t >> 3) : t;
}
// tile k of the lower triangle of T x T, in groups of G rows that walk over the columns together
__device__ __forceinline__ void lower_tile(int T, int G, int k, int& i, int& j) {
    int f = 0, size;
    for (;;) {
        size = min(G, T - f);
        const int all = size * f + size * (size + 1) / 2;
        if (k < all) break;
        k -= all;
        f += size;
    }
    if (k < size * f) {
        j = k / size, i = f + (k - j * size);
        return;
    }
    k -= size * f;
    j = 0;
    while (k >= size - j) k -= size - j, j++;
    i = f + j + k, j += f;
}
// tile k of TM x TN likewise
__device__ __forceinline__ void any_tile(int TM, int TN, int G, int k, int& i, int& j) {
    const int per = min(G, TM) * TN, f = k / per * min(G, TM), size = min(TM - f, G);
    k -= k / per * per;
    j = k / size, i = f + (k - j * size);
}
__device__ __forceinline__ int tiles_of(int x, int by) { return (x + by - 1) / by; }

struct Tile {
    int matrix, m0, n0, part, number;  // number: in its matrix
    bool none;  // a quarter beyond the matrix, or above the diagonal
};
template <int SIDE, bool LOWER> __device__ __forceinline__ Tile tile_at(const List& l, const Span& s, int t) {
    int id = number_of(s, t), part = 0;
    Tile r;
    r.part = 0;
    if (s.quarters) part = id & 3, id >>= 2;
    else if (s.splits > 1) r.part = id % s.splits, id /= s.splits;
    id += s.from;
    r.matrix = which(l, id);
    r.number = id - l.first[r.matrix];
    const Matrix& x = l.x[r.matrix];
    const int side = s.quarters ? 2 * SIDE : SIDE, M = LOWER ? x.pp() : x.mp, N = LOWER ? M : x.np;
    int i, j;
    if constexpr (LOWER) lower_tile(tiles_of(M, side), TOGETHER / side, id - l.first[r.matrix], i, j);
    else any_tile(tiles_of(M, side), tiles_of(N, side), TOGETHER / side, id - l.first[r.matrix], i, j);
    r.m0 = i * side + (part & 1) * SIDE, r.n0 = j * side + (part >> 1) * SIDE;
    r.none = r.m0 >= M || r.n0 >= N || (LOWER && r.m0 < r.n0);
    return r;
}

// A workgroup's tiles.  As long as they are of one matrix, and long enough for it, a tile's first
// stages are loaded under the last steps and the epilogue of the one before it.
template <int SIDE, bool LOWER, class Make> __device__ __forceinline__ void each_tile(const List& l, const Span& s, Make make) {
    for (int t = blockIdx.x; t < s.count; t += gridDim.x) {
        const Tile at = tile_at<SIDE, LOWER>(l, s, t);
        if (at.none) continue;
        make(l.x[at.matrix], at, [&](int steps, int NST) {
            return [&l, &s, &t, at, steps, NST](Place& p) {
                const int then = t + gridDim.x;
                if (steps <= NST || then >= s.count) return false;
                const Tile to = tile_at<SIDE, LOWER>(l, s, then);
                if (to.matrix != at.matrix || to.none || s.splits > 1) return false;
                t = then;
                p = Place{to.m0, to.n0, 0, steps};
                return true;
            };
        });
        __syncthreads();
    }
}

// a tile's values as float16 to its place and, where it lies below the diagonal, to the mirrored one: v[tn][tm] holds
// a lane's four consecutive columns of a row
template <class P> __device__ __forceinline__ void store_both(uint8_t* lds, const uint2 (&v)[P::TN][P::TM], uint16_t* c, int ld, int m0, int n0) {
    store_rows<P>(
        lds, [&](int tn, int tm) { return v[tn][tm]; },
        [&](int m, int n, const uint4& x) {
            if (m0 + m < ld && n0 + n < ld) *reinterpret_cast<uint4*>(c + (long)(m0 + m) * ld + n0 + n) = x;
        });
    if (m0 == n0) return;
    // the mirrored tile's rows are this one's columns: 16 at a time through the wave's part of LDS
    // (store_rows' part, so that no other wave is still in it)
    constexpr int CH = P::TM * 2, ROW = CH * 16, MINE = P::TN * 512 * (P::TN < 2 ? 2 : 1);
    static_assert(16 * ROW <= MINE && 8 * MINE <= P::EPILOGUE && CH <= 8, "tile");
    const int thread = thread_here(), lane = thread & 63, wave = thread >> 6, r16 = lane & 15, q = lane >> 4;
    uint8_t* mine = P::epilogue(lds) + wave * MINE;
    const int m = m0 + (wave / P::WN) * P::TM * 16 + 8 * (lane & (CH - 1)), nw = n0 + (wave % P::WN) * P::TN * 16;
#pragma unroll
    for (int tn = 0; tn < P::TN; tn++) {
#pragma unroll
        for (int tm = 0; tm < P::TM; tm++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int n = 4 * q + e, at = n * ROW + (((2 * tm + (r16 >> 3)) ^ ((n >> 1) & (CH - 1))) << 4) + 2 * (r16 & 7);
                const uint32_t w = e < 2 ? v[tn][tm].x : v[tn][tm].y;
                *reinterpret_cast<uint16_t*>(mine + at) = (uint16_t)(e & 1 ? w >> 16 : w);
            }
        wkv7::wave_lds_fence();
#pragma unroll
        for (int i = 0; i < 16 * CH / 64; i++) {
            const int r = i * (64 / CH) + lane / CH, n = nw + 16 * tn + r;
            const uint4 x = *reinterpret_cast<const uint4*>(mine + r * ROW + (((lane & (CH - 1)) ^ ((r >> 1) & (CH - 1))) << 4));
            if (m < ld && n < ld) *reinterpret_cast<uint4*>(c + (long)n * ld + m) = x;
        }
        wkv7::wave_lds_fence();
    }
}

// 64 x 64 tiles, for products of few tiles, whose steps are as long as their waits: four waves of 32 x 32 on each
// half of a step, their sums added at the end, and a step's fragments are read a whole step ahead, so that
// a step has one wait in which the reads, the matrix instructions and the barrier run together (353 x 1021:
// 0.25 us a step with eight waves on the tile, half steps one after the other).  Interface and layouts of Product;
// one tile a call.
template <int NST_, Lay LX_, Lay LY_> struct Slim {
    static constexpr int BM = 64, BN = 64, WM = 2, WN = 2, NST = NST_, TM = 2, TN = 2;
    static constexpr Lay LX = LX_, LY = LY_;
    static constexpr bool PERM = LX == RowN || LY == RowN;
    static constexpr int STAGE = (BM + BN) * BK * 2, EPILOGUE = 8 * TN * 512, SUMS = 4 * TM * TN * 1024;
    static constexpr int LDS = NST * STAGE, THREADS = 512, PIECES = 2;
    static_assert(SUMS + EPILOGUE <= LDS && NST >= 3, "stages");
    f32x4_t acc[TN][TM];

    __device__ static __forceinline__ uint8_t* epilogue(uint8_t* lds) { return lds + SUMS; }

    template <bool, class Next, class Done>
    __device__ __forceinline__ void go(uint8_t* lds, const Operand& X, const Operand& Y, Place at, Next, Done done) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave >> 2;
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
        Loader<LX, BM, PERM> lx(X, at.m0, at.step0 * BK, wave, lane);
        Loader<LY, BN, PERM> ly(Y, at.n0, at.step0 * BK, wave, lane);
        const Reader<LX, BM, PERM> rx((wave >> 1 & 1) * 32, lane);
        const Reader<LY, BN, PERM> ry((wave & 1) * 32, lane);
        auto load = [&](int stage, bool more) {
            lx.issue(lds0 + stage * STAGE, 0, wave);
            ly.issue(lds0 + stage * STAGE + BM * BK * 2, 0, wave);
            lx.advance(more), ly.advance(more);
        };
#pragma unroll
        for (int s = 0; s < NST; s++) load(s, s + 1 < at.steps);
#pragma unroll
        for (int tn = 0; tn < TN; tn++)
#pragma unroll
            for (int tm = 0; tm < TM; tm++) acc[tn][tm] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        struct Fragments {
            uint4 x[TM], y[TN];
        } a, b;
        auto read = [&](Fragments& f, int stage) {
#pragma unroll
            for (int i = 0; i < TM; i++) f.x[i] = rx.get(lds, stage * STAGE, i, half);
#pragma unroll
            for (int i = 0; i < TN; i++) f.y[i] = ry.get(lds, stage * STAGE + BM * BK * 2, i, half);
        };
        int cur = 0;
        auto step = [&](const Fragments& now, Fragments& then, int s) {
            // the next stage has landed, and every wave has this one's fragments
            wait_barrier<(NST - 2) * PIECES>();
            const int next = cur + 1 == NST ? 0 : cur + 1;
            load(cur, s + NST + 1 < at.steps);
            read(then, next);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int tn = 0; tn < TN; tn++)
#pragma unroll
                for (int tm = 0; tm < TM; tm++) acc[tn][tm] = wkv7::mma32h(acc[tn][tm], now.y[tn], now.x[tm]);
            cur = next;
        };
        wait_barrier<(NST - 1) * PIECES>();
        read(a, 0);
        int s = 0;
        for (; s + 1 < at.steps; s += 2) step(a, b, s), step(b, a, s + 1);
        if (s < at.steps) step(a, b, s);
        wkv7::vm_wait_n<0>();
        __syncthreads();
        f32x4_t* sums = reinterpret_cast<f32x4_t*>(lds) + (wave & 3) * (TM * TN * 64) + lane;
        if (half)
#pragma unroll
            for (int t = 0; t < TM * TN; t++) sums[64 * t] = acc[t / TM][t % TM];
        __syncthreads();
        if (half) return;
#pragma unroll
        for (int t = 0; t < TM * TN; t++) acc[t / TM][t % TM] += sums[64 * t];
        done(at);
    }
};

template <class P> __device__ __forceinline__ uint2 halves(const P& g, int tn, int tm) {
    const f32x4_t& a = g.acc[tn][tm];
    return make_uint2(half2_of(a[0], a[1]), half2_of(a[2], a[3]));
}

// A of the current X
template <class PW, class PT> __global__ __launch_bounds__(512) void gram(List l, Span s, int now) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[PW::LDS > PT::LDS ? PW::LDS : PT::LDS];
    each_tile<PW::BM, true>(l, s, [&](const Matrix& x, const Tile& at, auto more) {
        auto go = [&](auto tag, const Operand& o, int inner) {
            using P = decltype(tag);
            P g;
            const int all = inner / BK, each = (all + s.splits - 1) / s.splits, first = at.part * each;
            // (a part without steps makes one of zeros: from the last step, times nothing)
            g.template go<false>(lds, o, o, Place{at.m0, at.n0, min(first, all - 1), max(min(each, all - first), 0)}, more(each, P::NST), [&](const Place& t) {
                if (s.splits > 1) {
                    const int thread = thread_here();
                    f32x4_t* to = reinterpret_cast<f32x4_t*>(x.parts()) + ((long)at.number * s.splits + at.part) * (P::BM * P::BN / 4) + (thread >> 6) * (P::TM * P::TN * 64) + (thread & 63);
#pragma unroll
                    for (int tn = 0; tn < P::TN; tn++)
#pragma unroll
                        for (int tm = 0; tm < P::TM; tm++) to[(tn * P::TM + tm) * 64] = g.acc[tn][tm];
                    return;
                }
                uint2 v[P::TN][P::TM];
#pragma unroll
                for (int tn = 0; tn < P::TN; tn++)
#pragma unroll
                    for (int tm = 0; tm < P::TM; tm++) v[tn][tm] = halves(g, tn, tm);
                store_both<P>(lds, v, x.gram(), x.pp(), t.m0, t.n0);
            });
        };
        if (x.tall()) go(PT{}, Operand{x.hi(now), x.np, x.np, x.mp}, x.mp);
        else go(PW{}, Operand{x.hi(now), x.np, x.mp, x.np}, x.np);
    });
}

// A's parts added in order: a workgroup a tile, whose accumulators lie as gram's waves left them
template <class P> __global__ __launch_bounds__(256) void sum_gram(List l, Span s) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[P::LDS];
    const int splits = s.splits;
    s.splits = 1;
    const Tile at = tile_at<P::BM, true>(l, s, blockIdx.x);
    const Matrix& x = l.x[at.matrix];
    const f32x4_t* from = reinterpret_cast<const f32x4_t*>(x.parts()) + (long)at.number * splits * (P::BM * P::BN / 4) + (threadIdx.x >> 6) * (P::TM * P::TN * 64) + (threadIdx.x & 63);
    f32x4_t v[SPLITS][P::TM * P::TN];
#pragma unroll
    for (int k = 0; k < SPLITS; k++)
#pragma unroll
        for (int t = 0; t < P::TM * P::TN; t++) v[k][t] = from[(long)min(k, splits - 1) * (P::BM * P::BN / 4) + t * 64];
    P g;
#pragma unroll
    for (int t = 0; t < P::TM * P::TN; t++) {
        f32x4_t sum = v[0][t];
#pragma unroll
        for (int k = 1; k < SPLITS; k++) sum = k < splits ? sum + v[k][t] : sum;
        g.acc[t / P::TM][t % P::TM] = sum;
    }
    uint2 h[P::TN][P::TM];
#pragma unroll
    for (int tn = 0; tn < P::TN; tn++)
#pragma unroll
        for (int tm = 0; tm < P::TM; tm++) h[tn][tm] = halves(g, tn, tm);
    store_both<P>(lds, h, x.gram(), x.pp(), at.m0, at.n0);
}

// s^2 (a I + b A + c A^2) of A, with s^2 A in memory
template <class P> __global__ __launch_bounds__(512) void square(List l, Span s, float a, float b, float c) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[P::LDS];
    each_tile<P::BM, true>(l, s, [&](const Matrix& x, const Tile& at, auto more) {
        const int pp = x.pp();
        const Operand o{x.gram(), pp, pp, pp};
        P g;
        g.template go<false>(lds, o, o, Place{at.m0, at.n0, 0, pp / BK}, more(pp / BK, P::NST), [&](const Place& t) {
            const int thread = thread_here(), lane = thread & 63, wave = thread >> 6;
            const int m = t.m0 + (wave / P::WN) * P::TM * 16 + (lane & 15), n = t.n0 + (wave % P::WN) * P::TN * 16 + 4 * (lane >> 4);
            const float cs = c / (x.s * x.s), as = a * (x.s * x.s);
            const uint16_t* gram = x.gram();
            uint2 v[P::TN][P::TM];
#pragma unroll
            for (int tn = 0; tn < P::TN; tn++)
#pragma unroll
                for (int tm = 0; tm < P::TM; tm++)  // (places beyond the matrix are not stored: any valid ones)
                    v[tn][tm] = *reinterpret_cast<const uint2*>(gram + (long)min(m + 16 * tm, pp - 1) * pp + min(n + 16 * tn, pp - 4));
#pragma unroll
            for (int tn = 0; tn < P::TN; tn++)
#pragma unroll
                for (int tm = 0; tm < P::TM; tm++) {
                    const float2 x0 = floats_of(v[tn][tm].x), x1 = floats_of(v[tn][tm].y);
                    const f32x4_t& z = g.acc[tn][tm];
                    float y[4] = {b * x0.x + cs * z[0], b * x0.y + cs * z[1], b * x1.x + cs * z[2], b * x1.y + cs * z[3]};
                    if (t.m0 == t.n0) {
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] += m + 16 * tm == n + 16 * tn + e ? as : 0.f;
                    }
                    v[tn][tm] = make_uint2(half2_of(y[0], y[1]), half2_of(y[2], y[3]));
                }
            store_both<P>(lds, v, x.square(), pp, t.m0, t.n0);
        });
    });
}

// 16 (EACH = 2: 32) rows of a wave's tile of 16-bit values through its part of LDS, as store_rows
template <class P, int EACH, class Put> __device__ __forceinline__ void store_strip(uint8_t* lds, int t0, const uint2 (&v)[EACH][P::TN], Put put) {
    constexpr int CH = P::TN * 2, ROW = CH * 16;
    const int thread = thread_here(), lane = thread & 63, wave = thread >> 6, r16 = lane & 15, q = lane >> 4;
    uint8_t* mine = P::epilogue(lds) + wave * (EACH * 16 * ROW);
    const int c = lane & (CH - 1), m0 = (wave / P::WN) * P::TM * 16, n = (wave % P::WN) * P::TN * 16 + 8 * c;
#pragma unroll
    for (int t = 0; t < EACH; t++)
#pragma unroll
        for (int tn = 0; tn < P::TN; tn++)
            *reinterpret_cast<uint2*>(mine + (16 * t + r16) * ROW + (((2 * tn + (q >> 1)) ^ (r16 & (CH - 1))) << 4) + 8 * (q & 1)) = v[t][tn];
    wkv7::wave_lds_fence();
#pragma unroll
    for (int i = 0; i < EACH * 16 * CH / 64; i++) {
        const int r = i * (64 / CH) + lane / CH;
        put(m0 + 16 * t0 + r, n, *reinterpret_cast<const uint4*>(mine + r * ROW + ((c ^ (r & (CH - 1))) << 4)));
    }
    wkv7::wave_lds_fence();
}

// What an update makes of its sums: the next X in two halves, its first half alone (the step before the
// last, whose X goes nowhere but into products), or what the call is for.
enum Stage { BOTH, FIRST, LAST };
template <class P, Stage ST> __device__ __forceinline__ void update_done(P& g, uint8_t* lds, const Matrix& x, int now, float a, int tm0, int tn0) {
    constexpr int EACH = P::TN < 2 ? 2 : 1, STRIPS = P::TM / EACH;
    static_assert(P::TM % EACH == 0 && 8 * EACH * 16 * P::TN * 32 <= P::EPILOGUE, "tile");
    const int thread = thread_here(), lane = thread & 63, wave = thread >> 6;
    const int m = tm0 + (wave / P::WN) * P::TM * 16 + (lane & 15), n = tn0 + (wave % P::WN) * P::TN * 16 + 4 * (lane >> 4);
    const float by = 1.f / (x.s * x.s), al = a * (1.f / LO);
    uint2 o[2][EACH][P::TN];  // the second halves of a strip, and the next one's on their way
    auto fetch = [&](int s) {
#pragma unroll
        for (int t = 0; t < EACH; t++)
#pragma unroll
            for (int tn = 0; tn < P::TN; tn++)
                o[s & 1][t][tn] = *reinterpret_cast<const uint2*>(x.lo(now) + (long)min(m + 16 * (s * EACH + t), x.mp - 1) * x.np + min(n + 16 * tn, x.np - 4));
    };
    if constexpr (ST != LAST) fetch(0);
    auto put = [&](uint16_t* to) {
        return [&x, to, tm0, tn0](int i, int j, const uint4& v) {
            if (tm0 + i >= x.mp || tn0 + j >= x.np) return;
            u32x4* at = reinterpret_cast<u32x4*>(to + (long)(tm0 + i) * x.np + tn0 + j);
            // (a large X does not stay cached until the next step: streamed, four of 5120 x 5120 1026 -> 1002 us;
            // smaller ones are slower so, 768 x 768 23.9 -> 25.0)
            if constexpr (P::BM == 256) __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, at);
            else *at = u32x4{v.x, v.y, v.z, v.w};
        };
    };
#pragma unroll
    for (int s = 0; s < STRIPS; s++) {
        if constexpr (ST != LAST) {
            if (s + 1 < STRIPS) fetch(s + 1);
        }
        uint2 h[EACH][P::TN];
#pragma unroll
        for (int t = 0; t < EACH; t++)
#pragma unroll
            for (int tn = 0; tn < P::TN; tn++) {
                const f32x4_t& z = g.acc[tn][s * EACH + t];
                if constexpr (ST != LAST) {
                    uint2& lo = o[s & 1][t][tn];
                    const float2 o0 = floats_of(lo.x), o1 = floats_of(lo.y);
                    split(al * o0.x + by * z[0], al * o0.y + by * z[1], h[t][tn].x, lo.x);
                    split(al * o1.x + by * z[2], al * o1.y + by * z[3], h[t][tn].y, lo.y);
                } else {
                    const float is = by / x.s;
                    if (!x.momentum) {
                        h[t][tn] = make_uint2(f32x2_to_bf16x2(z[0] * is, z[1] * is), f32x2_to_bf16x2(z[2] * is, z[3] * is));
                        continue;
                    }
                    const int row = m + 16 * (s * EACH + t), col = n + 16 * tn;
                    if (row >= x.m || col >= x.n) continue;
                    float* p = static_cast<float*>(x.dst) + (long)row * x.n + col;
                    const float step = x.step * is;
                    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
                    if (col + 4 <= x.n) {
                        f4 v = *reinterpret_cast<f4*>(p);
                        for (int e = 0; e < 4; e++) v[e] = v[e] * x.keep - step * z[e];
                        *reinterpret_cast<f4*>(p) = v;
                    } else {
                        for (int e = 0; e < 4; e++)
                            if (col + e < x.n) p[e] = p[e] * x.keep - step * z[e];
                    }
                }
            }
        if constexpr (ST != LAST) {
            store_strip<P, EACH>(lds, s * EACH, h, put(x.hi(now ^ 1)));
            if constexpr (ST == BOTH) store_strip<P, EACH>(lds, s * EACH, o[s & 1], put(x.lo(now ^ 1)));
        } else if (!x.momentum) {
            store_strip<P, EACH>(lds, s * EACH, h, [&](int i, int j, const uint4& v) {
                const int row = tm0 + i, col = tn0 + j;
                if (row >= x.m || col >= x.n) return;
                uint16_t* to = static_cast<uint16_t*>(x.dst) + (long)row * x.n + col;
                typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
                if (col + 8 <= x.n) *reinterpret_cast<u4*>(to) = u4{v.x, v.y, v.z, v.w};
                else
                    for (int e = 0; e < 8 && col + e < x.n; e++) {
                        const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
                        to[e] = (uint16_t)(e & 1 ? w >> 16 : w);
                    }
            });
        }
    }
}

template <class PW, class PT, Stage ST> __global__ __launch_bounds__(512) void update(List l, Span s, Update u, int now, float a) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[PW::LDS > PT::LDS ? PW::LDS : PT::LDS];
    if (ST == LAST && skipped(u)) return;
    each_tile<PW::BM, false>(l, s, [&](const Matrix& x, const Tile& at, auto more) {
        const int pp = x.pp();
        const Operand B{x.square(), pp, pp, pp};
        auto go = [&](auto tag, const Operand& X, const Operand& Y) {
            using P = decltype(tag);
            P g;
            g.template go<false>(lds, X, Y, Place{at.m0, at.n0, 0, pp / BK}, more(pp / BK, P::NST),
                                 [&](const Place& t) { update_done<P, ST>(g, lds, x, now, a, t.m0, t.n0); });
        };
        // (B is symmetric: its rows serve as columns)
        if (x.tall()) go(PT{}, Operand{x.hi(now), x.np, x.mp, x.np}, B);
        else go(PW{}, B, Operand{x.hi(now), x.np, x.np, x.mp});
    });
}

// ------------------------------------------------------------------------------ short sides up to 128
// A list without longer ones takes one launch a step.  X^T lies in the workspace as [q][P] in its two halves, P = 64
// or 128.  A workgroup has a run of 16-row strips of it and a part of A from each of the run's
// workgroups before: it adds the parts, forms B in LDS, and its waves take two strips each,
//
//   Y = B X           B's rows from LDS, X's columns (the strips' rows) as they lie in memory
//
// whose halves go to memory and the first one to LDS as well, from where the waves make a part of the next A, each some
// tiles of its lower triangle, reading Y^T along its columns (LDS transpose reads).  Operands are
// float16 as above, here with X's second half in the product too; X and B are scaled apart, so that this half
// is no subnormal (X by 64, A by 64^2, B by 1024).  More workgroups shorten the strips' time and lengthen the
// parts'.  Four 2560 x 128 take 17 us a step: the launch 4, the parts 5.5, B 2, Y 1.5, its halves 2.7, the next A 1.
// 64 x 64 takes 21 us in all, 3.4 a step: each phase as long as its loads and LDS reads, X's halves to memory and back among them.
constexpr int SHORT = 128;
constexpr int ALONE = 16;  // strips that one workgroup takes: a list of such matrices takes one launch in all
constexpr float SX = 64.f, SB = 1024.f;

template <int P> struct Few {
    static constexpr int T = P / 16, TILES = T * (T + 1) / 2;
    static constexpr int LD = P + 8;         // 16 bytes more: rows on other banks
    static constexpr int HALVES = 8 / T;     // P = 64: two waves for a row of tiles, half of the strips each
    static constexpr int Y = P * LD * 2;     // behind B: Y^T of 16 strips,
    static constexpr int TURN = Y + 256 * LD * 2;        // the second halves of a strip for each wave
    static constexpr int LDS = TURN + 8 * 16 * LD * 2;
};
// tile (i, j) of a lower triangle, row after row
__device__ __forceinline__ constexpr int lower(int i, int j) { return i * (i + 1) / 2 + j; }
// P = 128: wave W's tiles of the next A, four or five, from rows W and 7 - W, whose column tiles (four, or five and the row's
// own) are all that the wave reads.  (A row of the triangle a wave takes 21.9 instead of 20.0 us a step; P = 64, with at most four
// tiles of a row and half of the strips a wave, stays so: 21.2 instead of 28.7 us for all.)
template <int W> struct Share {
    static constexpr int COUNT = W < 4 ? 5 : 4;
    static constexpr int i(int n) { return W < 4 || n >= W - 4 ? 7 - W : W; }
    static constexpr int j(int n) { return W < 4 ? n : n < W - 4 ? 5 + n : n - (W - 4); }
    static constexpr bool reads(int t) {
        for (int n = 0; n < COUNT; n++)
            if (i(n) == t || j(n) == t) return true;
        return false;
    }
};
template <class Go, int W = 0> __device__ __forceinline__ void share_of(int w, Go go) {
    if (w == W) go(Share<W>{});
    else if constexpr (W < 7) share_of<Go, W + 1>(w, go);
}

struct FewArgs {
    float a, b, c;
    int steps;
    int step;  // of this launch: 0 makes X_0 and its A, 1 .. steps the products
    const double* sums;
};

// A strip's elements in a matrix, for Y's accumulators d[t][e] (row 16 t + 4 q + e, column r16 of the strip).  Four
// consecutive ones at once where they are (a tall matrix of whole tiles); else by byte offsets from the strip's first
// element, behind the buffer for those that there are not.  (2^30 bytes: 128 rows of up to 2^21 elements.)
template <int T> struct Strip {
    static constexpr uint32_t BYTES = 1u << 30;
    uint8_t* base;
    uint32_t si, sj, first;
    int rows, size;  // rows: from this lane's first
    bool column, fours;
    __device__ __forceinline__ Strip(const void* m, bool tall, int p, int len, int j0, long ld, int size, int r16, int q) : size(size) {
        base = static_cast<uint8_t*>(const_cast<void*>(m)) + (tall ? j0 * ld : j0) * size;
        si = (tall ? 1 : (int)ld) * size, sj = (tall ? (int)ld : 1) * size;
        rows = p - 4 * q, column = j0 + r16 < len, fours = tall && p % 16 == 0;
        first = 4 * q * si + r16 * sj;
    }
    __device__ __forceinline__ uint32_t at(int i, int j) const { return column && 16 * i + j < rows ? first + (16 * i + j) * si : 2 * BYTES; }
    __device__ __forceinline__ void all(f32x4_t (&d)[T], bool fp32) const {
        const auto of = wkv7::make_rsrc(base, BYTES);
        if (fours) {
            const uint8_t* from = base + (column ? first : 0);  // (what is not there: the strip's first ones, and left out)
#pragma unroll
            for (int t = 0; t < T; t++) {
                const uint8_t* v = from + (16 * t < rows ? 16 * t * si : 0);
                if (fp32) {
                    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
                    const f4 y = *reinterpret_cast<const f4*>(v);
                    d[t] = f32x4_t{y[0], y[1], y[2], y[3]};
                } else {
                    typedef uint16_t u4 __attribute__((ext_vector_type(4), aligned(2)));
                    const u4 y = *reinterpret_cast<const u4*>(v);
                    d[t] = f32x4_t{bf16_to_f32(y[0]), bf16_to_f32(y[1]), bf16_to_f32(y[2]), bf16_to_f32(y[3])};
                }
            }
#pragma unroll
            for (int t = 0; t < T; t++)
                if (!column || 16 * t >= rows) d[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        } else {
#pragma unroll
            for (int t = 0; t < T; t++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    d[t][e] = fp32 ? __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(of, at(t, e), 0, 0))
                                   : bf16_to_f32(__builtin_amdgcn_raw_buffer_load_b16(of, at(t, e), 0, 0));
        }
    }
    __device__ __forceinline__ void put(const f32x4_t (&d)[T], bool fp32) const {
        const auto of = wkv7::make_rsrc(base, BYTES);
        if (fours) {
            if (!column) return;
#pragma unroll
            for (int t = 0; t < T; t++) {
                if (16 * t >= rows) break;
                uint8_t* v = base + first + 16 * t * si;
                if (fp32) {
                    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
                    *reinterpret_cast<f4*>(v) = f4{d[t][0], d[t][1], d[t][2], d[t][3]};
                } else {
                    typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(2)));
                    *reinterpret_cast<u2*>(v) = u2{f32x2_to_bf16x2(d[t][0], d[t][1]), f32x2_to_bf16x2(d[t][2], d[t][3])};
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < T; t++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (fp32) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(d[t][e]), of, at(t, e), 0, 0);
                    else __builtin_amdgcn_raw_buffer_store_b16(wkv7::f32_to_bf16(d[t][e]), of, at(t, e), 0, 0);
        }
    }
};

// (a workgroup's LDS alone: what goes to memory need not have arrived)
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// START: step 0, X_0 and its A from the call's matrix.  STEP: one of the others.  WHOLE: a workgroup a matrix, the momentum and
// its norm, then all steps, A's parts staying in LDS.
enum Part { START, STEP, WHOLE };
template <int P, Part KIND> __global__ __launch_bounds__(512) void few(List l, Update u, FewArgs f) {
    using F = Few<P>;
    constexpr int T = F::T, LD = F::LD;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[F::LDS];
    __shared__ double red[8];
    if (skipped(u)) return;
    uint16_t *mat = reinterpret_cast<uint16_t*>(lds), *yt = reinterpret_cast<uint16_t*>(lds + F::Y);  // A, then B; Y^T
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int k = which(l, blockIdx.x), groups = l.first[k + 1] - l.first[k], group = blockIdx.x - l.first[k];
    const Matrix& x = l.x[k];
    const bool tall = x.tall();
    const int p = tall ? x.n : x.m, len = tall ? x.m : x.n, strips = (len + 15) / 16, per = (strips + groups - 1) / groups;
    const int first = group * per, last = min(first + per, strips);
    uint16_t *xhi = x.ws, *xlo = xhi + (long)strips * 16 * P;                     // [q][P]
    float* parts = reinterpret_cast<float*>(xlo + (long)strips * 16 * P);         // [2][groups][HALVES][TILES][64][4]
    constexpr int PART = F::TILES * 256;
    float* near = reinterpret_cast<float*>(lds + F::Y);  // WHOLE: [HALVES][TILES][64][4]
    static_assert(F::HALVES * PART * 4 <= F::TURN - F::Y, "LDS");
    const float factor = u.result ? u.result[1] : u.factor;
    uint4 xh[2][P / 32], xl[2][P / 32];  // X's columns of this wave's two strips of those from s0 on, on their way while A is made
    auto load_x = [&](int s0) {
        const int lane = thread_here() & 63;
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int ks = 0; ks < P / 32; ks++) {  // (a wave without a second strip makes the last one again, and leaves it out)
                const int at = (16 * min(s0 + 2 * wave + s, last - 1) + (lane & 15)) * P + 32 * ks + 8 * (lane >> 4);
                xh[s][ks] = *reinterpret_cast<const uint4*>(xhi + at);
                xl[s][ks] = *reinterpret_cast<const uint4*>(xlo + at);
            }
    };

    auto make_step = [&](auto first_one, const int step) {
        constexpr bool start = decltype(first_one)::value;
        float by = 1.f / SB;
        f32x4_t d[2][T];
        // u in strips s0 + 2 wave and the next one; WHOLE: with the momentum's step and the sum of squares
        auto load_u = [&](int s0) {
            const int lane = thread_here() & 63, r16 = lane & 15, q = lane >> 4;
            double sum = 0;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const int j0 = 16 * min(s0 + 2 * wave + s, last - 1);
                const bool mine = s0 + 2 * wave + s < last;
                const Strip<T> src(x.src, tall, p, len, j0, x.ld, x.fp32 ? 4 : 2, r16, q);
                src.all(d[s], x.fp32);
                if (x.momentum) {
                    const Strip<T> mom(x.momentum, tall, p, len, j0, x.n, 4, r16, q);
                    f32x4_t m[T];
                    mom.all(m, true);
                    if constexpr (KIND == WHOLE) {
#pragma unroll
                        for (int t = 0; t < T; t++) m[t] = u.mu * m[t] + u.nu * (d[s][t] * factor);
                        if (mine) mom.put(m, true);
                    }
#pragma unroll
                    for (int t = 0; t < T; t++) d[s][t] = u.nesterov ? u.mu * m[t] + u.nu * (d[s][t] * factor) : m[t];
                }
                if (KIND == WHOLE && mine)
#pragma unroll
                    for (int t = 0; t < T; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sum += (double)d[s][t][e] * d[s][t][e];
            }
            return sum;
        };
        if constexpr (start) {  // the norm
            double sum = 0;
            if constexpr (KIND == WHOLE) sum = load_u(first);
            else
                for (int j = threadIdx.x; j < x.pieces; j += 512) sum += f.sums[x.piece0 + j];
            for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
            if ((threadIdx.x & 63) == 0) red[wave] = sum;
            __syncthreads();
            sum = 0;
            for (int w = 0; w < 8; w++) sum += red[w];
            const double norm = sqrt(sum);
            by = (float)(SX / (norm < u.eps ? (double)u.eps : norm));
        } else {  // A's parts in order, A, B
            const int count = groups * F::HALVES;
            constexpr int MINE = (F::TILES * 64 + 511) / 512;
            f32x4_t s[MINE];
#pragma unroll
            for (int r = 0; r < MINE; r++) s[r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if constexpr (KIND == WHOLE) {
                wkv7::vm_wait_n<0>();  // (this wave's X is written)
                load_x(first);
#pragma unroll
                for (int h = 0; h < F::HALVES; h++)
#pragma unroll
                    for (int r = 0; r < MINE; r++)
                        s[r] += *reinterpret_cast<const f32x4_t*>(near + h * PART + 4 * threadIdx.x + (threadIdx.x + 512 * r < F::TILES * 64 ? 2048 * r : 0));
            } else {  // (a batch in flight, added one after the other)
                constexpr int BATCH = 10;
                const float* from = parts + (long)((step - 1) & 1) * count * PART + 4 * threadIdx.x;
                for (int g0 = 0; g0 < count; g0 += BATCH) {
                    f32x4_t v[BATCH][MINE];
#pragma unroll
                    for (int g = 0; g < BATCH; g++)
#pragma unroll
                        for (int r = 0; r < MINE; r++)
                            v[g][r] = *reinterpret_cast<const f32x4_t*>(from + (long)min(g0 + g, count - 1) * PART + (threadIdx.x + 512 * r < F::TILES * 64 ? 2048 * r : 0));
#pragma unroll
                    for (int g = 0; g < BATCH; g++)
#pragma unroll
                        for (int r = 0; r < MINE; r++) {
                            if (g0 + g >= count) break;
                            asm volatile("");  // (a branch: selects would cost as much as the sums)
                            s[r] += v[g][r];
                        }
                }
                load_x(first);
            }
#pragma unroll
            for (int r = 0; r < MINE; r++) {
                const int tile = wave + 8 * r, rr = threadIdx.x & 15, qq = threadIdx.x >> 4 & 3;
                if (tile >= F::TILES) break;
                int i = 0;
#pragma unroll
                for (int n = 1; n < T; n++) i += tile >= lower(n, 0);
                const int j = tile - lower(i, 0), row = 16 * i + 4 * qq, col = 16 * j + rr;
                const uint2 h = make_uint2(half2_of(s[r][0], s[r][1]), half2_of(s[r][2], s[r][3]));
                *reinterpret_cast<uint2*>(mat + col * LD + row) = h;
                if (i != j) {
                    mat[row * LD + col] = (uint16_t)h.x, mat[(row + 1) * LD + col] = (uint16_t)(h.x >> 16);
                    mat[(row + 2) * LD + col] = (uint16_t)h.y, mat[(row + 3) * LD + col] = (uint16_t)(h.y >> 16);
                }
            }
            lds_barrier();
            // wave w: rows 16 (w % T) .., of P = 64 half of the columns each
            const int lane = thread_here() & 63, r16 = lane & 15, q = lane >> 4;
            constexpr int N = T / F::HALVES;
            const int ti = wave % T, tj0 = wave / T * N;
            f32x4_t acc[N];
#pragma unroll
            for (int n = 0; n < N; n++) acc[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < P / 32; ks++) {
                const uint4 av = *reinterpret_cast<const uint4*>(mat + (16 * ti + r16) * LD + 32 * ks + 8 * q);
#pragma unroll
                for (int n = 0; n < N; n++)
                    acc[n] = wkv7::mma32h(acc[n], av, *reinterpret_cast<const uint4*>(mat + (16 * (tj0 + n) + r16) * LD + 32 * ks + 8 * q));
            }
            const float fa = f.a * SB, fb = f.b * (SB / (SX * SX)), fc = f.c * (SB / (SX * SX * SX * SX));
            uint2 b[N];
#pragma unroll
            for (int n = 0; n < N; n++) {  // (row 16 ti + 4 q + e, column 16 (tj0 + n) + r16; A from the mirrored place)
                const int row = 16 * ti + 4 * q, col = 16 * (tj0 + n) + r16;
                const uint2 av = *reinterpret_cast<const uint2*>(mat + col * LD + row);
                const float2 a0 = floats_of(av.x), a1 = floats_of(av.y);
                const float y[4] = {fb * a0.x + fc * acc[n][0], fb * a0.y + fc * acc[n][1], fb * a1.x + fc * acc[n][2], fb * a1.y + fc * acc[n][3]};
                b[n] = make_uint2(half2_of(y[0] + (row == col ? fa : 0.f), y[1] + (row + 1 == col ? fa : 0.f)),
                                  half2_of(y[2] + (row + 2 == col ? fa : 0.f), y[3] + (row + 3 == col ? fa : 0.f)));
            }
            lds_barrier();
#pragma unroll
            for (int n = 0; n < N; n++) *reinterpret_cast<uint2*>(mat + (16 * (tj0 + n) + r16) * LD + 16 * ti + 4 * q) = b[n];
            lds_barrier();
        }
        // 16 strips at a time
        const int row = wave % T, half = wave / T;  // of the next A's tiles
        constexpr int MOST = T == 8 ? 5 : 4;
        f32x4_t gram[MOST];
#pragma unroll
        for (int t = 0; t < MOST; t++) gram[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        for (int s0 = first; s0 < last; s0 += 16) {
            const int lane = thread_here() & 63, r16 = lane & 15, q = lane >> 4;
            const int strip = s0 + 2 * wave, have = min(last - strip, 2);
            auto make = [&] {
            if constexpr (start) {
                if constexpr (KIND == START) load_u(s0);
            } else {
#pragma unroll
                for (int t = 0; t < T; t++) {
                    d[0][t] = d[1][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < P / 32; ks++) {
                        const uint4 b = *reinterpret_cast<const uint4*>(mat + (16 * t + r16) * LD + 32 * ks + 8 * q);
#pragma unroll
                        for (int s = 0; s < 2; s++) {
                            d[s][t] = wkv7::mma32h(d[s][t], b, xh[s][ks]);
                            d[s][t] = wkv7::mma32h(d[s][t], b, xl[s][ks]);
                        }
                    }
                }
                if (step == f.steps) {
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        if (s >= have) break;
                        const Strip<T> dst(x.dst, tall, p, len, 16 * (strip + s), x.n, x.momentum ? 4 : 2, r16, q);
                        const float to = by / SX, step_by = x.step * to;
                        if (x.momentum) {
                            f32x4_t w[T];
                            dst.all(w, true);
#pragma unroll
                            for (int t = 0; t < T; t++) d[s][t] = w[t] * x.keep - step_by * d[s][t];
                        } else {
#pragma unroll
                            for (int t = 0; t < T; t++) d[s][t] *= to;
                        }
                        dst.put(d[s], x.momentum);
                    }
                    return;
                }
            }
            // whole rows of X^T to memory through LDS, the first halves staying there
            uint16_t* turn = reinterpret_cast<uint16_t*>(lds + F::TURN) + wave * 16 * LD;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                uint16_t* mine = yt + (32 * wave + 16 * s) * LD;
#pragma unroll
                for (int t = 0; t < T; t++) {
                    uint2 h, o;
                    split<1>(d[s][t][0] * by, d[s][t][1] * by, h.x, o.x);
                    split<1>(d[s][t][2] * by, d[s][t][3] * by, h.y, o.y);
                    if (s >= have) h = make_uint2(0, 0);
                    *reinterpret_cast<uint2*>(mine + r16 * LD + 16 * t + 4 * q) = h;
                    *reinterpret_cast<uint2*>(turn + r16 * LD + 16 * t + 4 * q) = o;
                }
                wkv7::wave_lds_fence();
                constexpr int CH = P / 8;
#pragma unroll
                for (int v = 0; v < 16 * CH / 64; v++) {
                    const int j = (64 * v + lane) / CH, col = 8 * ((64 * v + lane) % CH), at = (16 * (strip + s) + j) * P + col;
                    const uint4 h = *reinterpret_cast<const uint4*>(mine + j * LD + col), o = *reinterpret_cast<const uint4*>(turn + j * LD + col);
                    if (s < have) {
                        *reinterpret_cast<uint4*>(xhi + at) = h;
                        *reinterpret_cast<uint4*>(xlo + at) = o;
                    }
                }
                wkv7::wave_lds_fence();
            }
            };
            if (s0 > first) lds_barrier();  // (the strips before are still read)
            if (have > 0) make();
            if (!start && s0 + 16 < last) load_x(s0 + 16);
            if (!start && step == f.steps) continue;
            lds_barrier();
            // (lane: rows 4 q + (r16 >> 2) and 16 behind of 32 of Y^T, four columns, turned by the read)
            const uint16_t* at = yt + (4 * q + (r16 >> 2)) * LD + 4 * (r16 & 3);
            const int pairs = (min(last - s0, 16) + 1) / 2;  // (of strips: rows beyond the last one's are zero)
            auto frag = [&](int ks, int t) {
                const uint2 lo = wkv7::tr_at(at + 32 * ks * LD + 16 * t), hi = wkv7::tr_at(at + (32 * ks + 16) * LD + 16 * t);
                return make_uint4(lo.x, lo.y, hi.x, hi.y);
            };
            if constexpr (T == 8) {
                share_of(row, [&](auto mine) {
                    using S = decltype(mine);
                    for (int ks = 0; ks < pairs; ks++) {
                        uint4 y[T];
#pragma unroll
                        for (int t = 0; t < T; t++)
                            if (S::reads(t)) y[t] = frag(ks, t);
#pragma unroll
                        for (int n = 0; n < S::COUNT; n++) gram[n] = wkv7::mma32h(gram[n], y[S::i(n)], y[S::j(n)]);
                    }
                });
            } else {
                for (int ks = half; ks < pairs; ks += F::HALVES) {
                    const uint4 a = frag(ks, row);
#pragma unroll
                    for (int t = 0; t < T; t++) gram[t] = wkv7::mma32h(gram[t], a, frag(ks, t));  // (all reads at once; those above the diagonal are left out)
                }
            }
        }
        if (!start && step == f.steps) return;
        f32x4_t* to;
        if constexpr (KIND == WHOLE) {
            lds_barrier();  // (Y^T, in whose place the parts go, is still read)
            to = reinterpret_cast<f32x4_t*>(near + half * PART) + (thread_here() & 63);
        } else {
            to = reinterpret_cast<f32x4_t*>(parts + (((long)(step & 1) * groups + group) * F::HALVES + half) * PART) + (thread_here() & 63);
        }
        if constexpr (T == 8) {
            share_of(row, [&](auto mine) {
                using S = decltype(mine);
#pragma unroll
                for (int n = 0; n < S::COUNT; n++) to[lower(S::i(n), S::j(n)) * 64] = gram[n];
            });
        } else {
#pragma unroll
            for (int t = 0; t < T; t++) {
                if (t > row) break;
                to[lower(row, t) * 64] = gram[t];
            }
        }
        if constexpr (KIND == WHOLE) lds_barrier();
    };
    if constexpr (KIND != STEP) make_step(std::true_type{}, 0);
    if constexpr (KIND == STEP) make_step(std::false_type{}, f.step);
    if constexpr (KIND == WHOLE)
        for (int step = 1; step <= f.steps; step++) make_step(std::false_type{}, step);
}

// ------------------------------------------------------------------------------ host
static long up(long x, long to) { return (x + to - 1) / to * to; }
static long ceil_div(long x, long y) { return (x + y - 1) / y; }

template <int BM, int WM, int WN, int NST> struct Shape {
    using KK = Product<BM, BM, WM, WN, NST, RowK, RowK, true>;
    using NN = Product<BM, BM, WM, WN, NST, RowN, RowN, true>;
    using KN = Product<BM, BM, WM, WN, NST, RowK, RowN, true>;
};
using Large = Shape<256, 4, 2, 2>;
using Middle = Shape<128, 4, 2, 2>;
using Deep = Shape<128, 4, 2, 4>;
struct Small {
    using KK = Slim<4, RowK, RowK>;
    using NN = Slim<4, RowN, RowN>;
    using KN = Slim<4, RowK, RowN>;
};
// Side, workgroups on a CU; us of a step of 64 along the contraction where few workgroups run and where all do
// (they share the caches and the power), of the rest of a tile, and what a square's or an update's epilogue adds.
// From squares of 256 .. 4096, 192, 352 and 512 x 5120 and 4096, each made in all four: Gram matrices of
// 768 x 768 take 23, 12, 11 and 7 us, of 2048 x 2048 44, 24, 19 and 23, of 192 x 5120 89, 48, 33 and 18, of four of
// 5120 x 5120 513 in tiles of 256 with the last round in quarters; updates of 2048 x 2048 52, 31, 27 and 43.
struct Cost {
    int side, per_cu;
    double few, full, rest, epilogue;
};
constexpr double LAUNCH = 4;  // us of one more launch
constexpr Cost COSTS[] = {{256, 1, 1.1, 1.75, 7, 8}, {128, 2, .56, 1.15, 5, 2}, {128, 1, .36, .6, 5, 2}, {64, 2, .17, .52, 4.2, 1}};
constexpr int SHAPES = sizeof COSTS / sizeof *COSTS;

static int device_cus() {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 256;
    return n > 0 ? n : 256;
}

constexpr size_t MOST = 4ull << 30;  // bytes of the matrices of a launch together, if it has more than one

// A matrix of a list of short sides: strips, and workgroups where `matrices` share the card: two
// strips for each wave, more where the parts of so many workgroups take longer.
static bool is_short(int m, int n) { return (m < n ? m : n) <= SHORT; }
static long strips_of(const Matrix& x) { return ceil_div(x.m < x.n ? x.n : x.m, 16); }
static long groups_of(const Matrix& x, int matrices) {
    const long strips = strips_of(x), share = 256 / matrices > 1 ? 256 / matrices : 1;
    if (strips <= ALONE) return 1;
    long n = 1;
    while (n * n < 2 * strips) n++;
    const long pairs = ceil_div(strips, 16);
    n = n < pairs ? n : pairs, n = n < share ? n : share;
    return ceil_div(strips, ceil_div(strips, n));  // (none without strips)
}
static size_t short_bytes(const Matrix& x) {  // (beside any others)
    return up(strips_of(x) * 16 * SHORT * 4 + 2 * groups_of(x, 1) * Few<SHORT>::TILES * 1024, 256);  // (P = 64: two parts of 10 KB each, less)
}
// A's contraction is split where its tiles of 64 leave CUs idle: up to this many tiles
constexpr long SPLIT_TILES = 128;
static bool splits(const Matrix& x) {
    const long p = x.pp() / 64;
    return p * (p + 1) / 2 <= SPLIT_TILES;
}
static size_t bytes_of(const Matrix& x) {
    const size_t p = x.pp() / 64;
    return 2 * (4 * (size_t)x.mp * x.np + 2 * (size_t)x.pp() * x.pp()) + (splits(x) ? p * (p + 1) / 2 * SPLITS * 64 * 64 * 4 : 0);
}

static Matrix matrix(int m, int n) {
    Matrix x{};
    x.m = m, x.n = n, x.mp = (int)up(m, BK), x.np = (int)up(n, BK);
    const int p = m < n ? m : n;
    x.s = 1.f;
    while (x.s < 32.f && 4.f * x.s * x.s <= (float)p) x.s *= 2.f;  // (a s^2 stays far below 65504)
    // (few elements: every load at once rather than few workgroups; many: at most 4096 sums, which every workgroup of X_0 adds)
    const long many = ceil_div((long)m * n, 4096l * PIECE);
    x.each = (long)m * n <= 1 << 20 ? 1 : many < 4 ? 4 : (int)many;
    x.pieces = (int)ceil_div((long)m * ceil_div(n, 8), PIECE / 8 * x.each);
    x.ld = n;
    return x;
}

// Whether a call has short sides alone (beside longer ones they take part in the products' launches).
template <class Get> static bool only_short(int count, Get get) {
    for (int i = 0; i < count; i++) {
        const Matrix x = get(i);
        if (x.m && x.n && !is_short(x.m, x.n)) return false;
    }
    return true;
}
// The list's matrices from `next` on that one set of launches takes.
template <class Get> static bool take(int count, int& next, Get get, bool all_short, List& l, size_t& bytes, long& pieces) {
    l.count = 0;
    bytes = 0, pieces = 0;
    while (next < count && l.count < MAX) {
        Matrix x = get(next);
        if (x.m && x.n) {
            const size_t size = all_short ? short_bytes(x) : bytes_of(x);
            if (l.count && bytes + size > MOST) break;
            x.piece0 = (int)pieces;
            pieces += x.pieces;
            bytes += size;
            l.x[l.count++] = x;
        }
        next++;
    }
    return l.count > 0;
}
static size_t sums_bytes(long pieces) { return up(pieces * sizeof(double), 256); }

template <class Get> static size_t workspace(int count, Get get) {
    size_t most = 0, bytes;
    long pieces;
    int next = 0;
    List l;
    const bool all_short = only_short(count, get);
    while (take(count, next, get, all_short, l, bytes, pieces)) most = most > bytes + sums_bytes(pieces) ? most : bytes + sums_bytes(pieces);
    return most;
}

// tiles of matrix x in a product: the lower triangle of the Gram matrix or its square, or all of X
static long tiles(const Matrix& x, bool lower, int side) {
    const long p = ceil_div(x.pp(), side);
    return lower ? p * (p + 1) / 2 : ceil_div(x.mp, side) * ceil_div(x.np, side);
}
// How a product of the whole list is made: tiles of 256 where they fill the CUs, smaller ones (twice the
// operands' traffic for each halving) where there are few; a last round that would fill few CUs in
// quarters of its tiles.
struct Way {
    int shape;
    bool quarters;   // the tiles behind the last full round, in the next shape
    int splits = 1;  // of every tile's contraction, added by a launch of its own
};
static Way way(const List& l, bool lower, bool gram, int cus) {
    // us of `count` of the list's tiles in a shape, as many as there are slots at once
    auto round = [&](const Cost& c, double count, int splits = 1) {
        const double load = count / (cus * c.per_cu), step = c.few + (c.full - c.few) * (load < 1 ? load : 1);
        double sum = 0, n = 0, longest = 0;
        for (int k = 0; k < l.count; k++) {
            const Matrix& x = l.x[k];
            const double w = (double)tiles(x, lower, c.side), t = c.rest + (gram ? 0 : c.epilogue) + step * ceil((gram ? (x.tall() ? x.mp : x.np) : x.pp()) / BK / (double)splits);
            sum += w * t, n += w;
            longest = longest > t ? longest : t;
        }
        return load < 1 ? longest : sum / n;
    };
    Way best{0, false};
    double least = 0;
    for (int i = 0; i < SHAPES; i++) {
        const Cost& c = COSTS[i];
        double n = 0;
        for (int k = 0; k < l.count; k++) n += (double)tiles(l.x[k], lower, c.side);
        const double slots = cus * c.per_cu, full = floor(n / slots), left = n - full * slots, rounds = full ? full * round(c, slots) : 0;
        const double us = rounds + (left ? round(c, left) : 0);
        if (i == 0 || us < least) least = us, best = Way{i, false};
        if (i == 0 && full && left) {
            const double q = cus * COSTS[1].per_cu, many = floor(4 * left / q), few = 4 * left - many * q;
            const double in4 = rounds + LAUNCH + (many ? many * round(COSTS[1], q) : 0) + (few ? round(COSTS[1], few) : 0);
            if (in4 < least) least = in4, best = Way{i, true};
        }
        if (i == SHAPES - 1 && gram) {
            bool all = true;
            for (int k = 0; k < l.count; k++) all &= splits(l.x[k]);
            for (int k = 2; all && k <= SPLITS && n * k <= slots; k++) {
                const double in = round(c, n * k, k) + LAUNCH + 2;
                if (in < least) least = in, best = Way{i, false, k};
            }
        }
    }
    return best;
}

template <class Set> static unsigned prefix(List& l, Set groups) {
    long at = 0;
    for (int k = 0; k < l.count; k++) {
        l.first[k] = (int)at;
        at += groups(l.x[k]);
    }
    l.first[l.count] = (int)at;
    return (unsigned)at;
}

static void run(List& l, const Update& u, const theseus_newton_schulz* ns, bool all_short, uint8_t* ws, long pieces, hipStream_t st) {
    double* sums = reinterpret_cast<double*>(ws);
    uint8_t* at = ws + sums_bytes(pieces);
    for (int k = 0; k < l.count; k++) {
        l.x[k].ws = reinterpret_cast<uint16_t*>(at);
        at += all_short ? short_bytes(l.x[k]) : bytes_of(l.x[k]);
    }
    const int cus = device_cus();
    int longest = 0;
    bool whole = all_short;
    for (int k = 0; k < l.count; k++) {
        const int p = l.x[k].m < l.x[k].n ? l.x[k].m : l.x[k].n;
        longest = longest > p ? longest : p;
        whole &= strips_of(l.x[k]) <= ALONE;
    }
    if (!whole) momentum_norm<<<prefix(l, [](const Matrix& x) { return (long)x.pieces; }), 256, 0, st>>>(l, u, sums);
    if (all_short) {
        const unsigned n = prefix(l, [&](const Matrix& x) { return groups_of(x, l.count); });
        auto go = [&](auto P) {
            constexpr int side = decltype(P)::value;
            FewArgs f{ns->a, ns->b, ns->c, ns->steps, 0, sums};
            if (whole) {
                few<side, WHOLE><<<n, 512, 0, st>>>(l, u, f);
                return;
            }
            few<side, START><<<n, 512, 0, st>>>(l, u, f);
            for (f.step = 1; f.step <= ns->steps; f.step++) few<side, STEP><<<n, 512, 0, st>>>(l, u, f);
        };
        if (longest <= 64) go(std::integral_constant<int, 64>{});
        else go(std::integral_constant<int, SHORT>{});
        return;
    }
    const unsigned scale = prefix(l, [](const Matrix& x) { return ceil_div((long)x.mp * x.np, PIECE * x.each); });
    scale_split<<<scale, 256, 0, st>>>(l, u, sums);
    const Way wg = way(l, true, true, cus), ws2 = way(l, true, false, cus), wu = way(l, false, false, cus);
    // one product: go(shape, workgroups, span)
    auto with = [&](const Way& w, bool lower, auto go) {
        const Cost& c = COSTS[w.shape];
        const int total = (int)prefix(l, [&](const Matrix& x) { return tiles(x, lower, c.side); });
        auto part = [&](int shape, const Span& s) {
            const int slots = cus * COSTS[shape].per_cu / 8 * 8;
            const unsigned n = s.count < slots || slots == 0 ? s.count : slots;
            if (shape == 0) go(Large{}, n, s);
            else if (shape == 1) go(Middle{}, n, s);
            else if (shape == 2) go(Deep{}, n, s);
            else go(Small{}, n, s);
        };
        const int slots = cus * c.per_cu, full = w.quarters ? total / slots * slots : total;
        part(w.shape, Span{0, full * w.splits, false, w.splits});
        if (full < total) part(w.shape + 1, Span{full, 4 * (total - full), true});
    };
    for (int i = 0; i < ns->steps; i++) {
        const int now = i & 1;
        with(wg, true, [&](auto shape, unsigned n, const Span& s) {
            using S = decltype(shape);
            gram<typename S::KK, typename S::NN><<<n, 512, 0, st>>>(l, s, now);
            if constexpr (std::is_same_v<S, Small>)
                if (s.splits > 1) sum_gram<typename S::KK><<<(unsigned)(s.count / s.splits), 256, 0, st>>>(l, Span{0, s.count / s.splits, false, s.splits});
        });
        with(ws2, true, [&](auto shape, unsigned n, const Span& s) {
            using S = decltype(shape);
            square<typename S::KK><<<n, 512, 0, st>>>(l, s, ns->a, ns->b, ns->c);
        });
        with(wu, false, [&](auto shape, unsigned n, const Span& s) {
            using S = decltype(shape);
            if (i + 1 == ns->steps) update<typename S::KN, typename S::KK, LAST><<<n, 512, 0, st>>>(l, s, u, now, ns->a);
            else if (i + 2 == ns->steps) update<typename S::KN, typename S::KK, FIRST><<<n, 512, 0, st>>>(l, s, u, now, ns->a);
            else update<typename S::KN, typename S::KK, BOTH><<<n, 512, 0, st>>>(l, s, u, now, ns->a);
        });
    }
}

static int check(const theseus_newton_schulz* ns) {
    if (!ns) return THESEUS_WKV7_ERR_NULL;
    if (ns->steps < 1 || ns->steps > 100 || !isfinite(ns->a) || !isfinite(ns->b) || !isfinite(ns->c) || !(ns->eps >= 0.f) || !isfinite(ns->eps))
        return THESEUS_WKV7_ERR_SHAPE;
    return THESEUS_WKV7_OK;
}
static float eps_of(const theseus_newton_schulz* ns) { return ns->eps > 1e-30f ? ns->eps : 1e-30f; }  // (64 over it is finite)
constexpr long long MAX_STRIDE = 1ll << 21;  // elements from row to row, in 32-bit byte offsets within a strip
static bool fits(long long m, long long n) { return m >= 0 && n >= 0 && m <= 1 << 17 && n <= 1 << 17; }

static Matrix get_orth(const theseus_orthogonalize_matrix& s) {
    Matrix x = matrix(s.rows, s.cols);
    x.src = s.x, x.ld = s.rows > 1 ? s.row_stride : s.cols, x.dst = s.out, x.fp32 = s.dtype == THESEUS_MUON_FP32;
    return x;
}
static Matrix get_muon(const theseus_muon_matrix& s) {
    Matrix x = matrix(s.rows, s.cols);
    x.src = s.grad, x.momentum = s.momentum, x.dst = s.param, x.keep = s.keep, x.step = s.step, x.fp32 = 1;
    return x;
}
static int check(const theseus_orthogonalize_matrix* ms, int count) {
    if (count < 0) return THESEUS_WKV7_ERR_SHAPE;
    if (count && !ms) return THESEUS_WKV7_ERR_NULL;
    for (int i = 0; i < count; i++) {
        const theseus_orthogonalize_matrix& s = ms[i];
        if (!fits(s.rows, s.cols) || (s.rows > 1 && (s.row_stride < s.cols || s.row_stride > MAX_STRIDE))) return THESEUS_WKV7_ERR_SHAPE;
        if (s.dtype != THESEUS_MUON_BF16 && s.dtype != THESEUS_MUON_FP32) return THESEUS_WKV7_ERR_DTYPE;
        if (s.rows && s.cols && (!s.x || !s.out)) return THESEUS_WKV7_ERR_NULL;
    }
    return THESEUS_WKV7_OK;
}
static int check(const theseus_muon_matrix* ms, int count) {
    if (count < 0) return THESEUS_WKV7_ERR_SHAPE;
    if (count && !ms) return THESEUS_WKV7_ERR_NULL;
    for (int i = 0; i < count; i++) {
        const theseus_muon_matrix& s = ms[i];
        if (!fits(s.rows, s.cols)) return THESEUS_WKV7_ERR_SHAPE;
        if (s.rows && s.cols && (!s.param || !s.grad || !s.momentum)) return THESEUS_WKV7_ERR_NULL;
    }
    return THESEUS_WKV7_OK;
}

// The norm pass over the gradients, a launch's tensors at a time; partial == nullptr: its doubles alone.
static long long norm_pass(const theseus_muon_matrix* ms, int count, double* partial, hipStream_t st) {
    theseus_adamw_tensor t[MAX];
    long long chunks = 0;
    for (int i = 0; i < count; i += MAX) {
        const int n = count - i < MAX ? count - i : MAX;
        for (int k = 0; k < n; k++) {
            t[k] = theseus_adamw_tensor{};
            t[k].grad = ms[i + k].grad, t[k].numel = (long long)ms[i + k].rows * ms[i + k].cols;
            if (!partial) chunks += (t[k].numel + THESEUS_ADAMW_CHUNK - 1) / THESEUS_ADAMW_CHUNK;
        }
        if (partial) optim::launch_sumsq(t, n, chunks, 0, partial, st);
    }
    return chunks;
}

}  // namespace muon

extern "C" {

size_t theseus_orthogonalize_workspace_size(const theseus_orthogonalize_matrix* ms, int count) {
    if (muon::check(ms, count)) return 0;
    return muon::workspace(count, [&](int i) { return muon::get_orth(ms[i]); });
}

int theseus_orthogonalize(const theseus_orthogonalize_matrix* ms, int count, const theseus_newton_schulz* ns, void* workspace,
                          size_t workspace_bytes, hipStream_t stream) {
    if (int e = muon::check(ns)) return e;
    if (int e = muon::check(ms, count)) return e;
    auto get = [&](int i) { return muon::get_orth(ms[i]); };
    const size_t need = muon::workspace(count, get);
    if (!need) return THESEUS_WKV7_OK;
    if (!workspace || workspace_bytes < need) return THESEUS_WKV7_ERR_WORKSPACE;
    const muon::Update u{0.f, 1.f, 0, 1.f, nullptr, 0, muon::eps_of(ns)};
    muon::List l;
    size_t bytes;
    long pieces;
    int next = 0;
    const bool all_short = muon::only_short(count, get);
    while (muon::take(count, next, get, all_short, l, bytes, pieces)) muon::run(l, u, ns, all_short, static_cast<uint8_t*>(workspace), pieces, stream);
    return hipGetLastError() == hipSuccess ? THESEUS_WKV7_OK : THESEUS_WKV7_ERR_LAUNCH;
}

size_t theseus_muon_workspace_size(const theseus_muon_matrix* ms, int count) {
    if (muon::check(ms, count)) return 0;
    const size_t norm = (size_t)muon::norm_pass(ms, count, nullptr, nullptr) * sizeof(double), step = muon::workspace(count, [&](int i) { return muon::get_muon(ms[i]); });
    return norm > step ? norm : step;
}

int theseus_muon_step(const theseus_muon_matrix* ms, int count, const theseus_newton_schulz* ns, double momentum, int nesterov,
                      float grad_scale, float max_norm, int skip_nonfinite, float* result, void* workspace, size_t workspace_bytes,
                      hipStream_t stream) {
    if (int e = muon::check(ns)) return e;
    if (int e = muon::check(ms, count)) return e;
    const bool norm = max_norm >= 0.f;
    if (norm && !result) return THESEUS_WKV7_ERR_NULL;
    const size_t need = theseus_muon_workspace_size(ms, count);
    if (!need && !norm) return THESEUS_WKV7_OK;
    if (need && (!workspace || workspace_bytes < need)) return THESEUS_WKV7_ERR_WORKSPACE;
    if (result) {  // (written without a norm too: a caller may read it)
        double* partial = norm ? static_cast<double*>(workspace) : nullptr;
        optim::launch_norm(partial, norm ? muon::norm_pass(ms, count, partial, stream) : 0, grad_scale, max_norm, result, stream);
    }
    const muon::Update u{(float)momentum, (float)(1.0 - momentum), nesterov, grad_scale, norm ? result : nullptr, skip_nonfinite, muon::eps_of(ns)};
    auto get = [&](int i) { return muon::get_muon(ms[i]); };
    muon::List l;
    size_t bytes;
    long pieces;
    int next = 0;
    const bool all_short = muon::only_short(count, get);
    while (muon::take(count, next, get, all_short, l, bytes, pieces)) muon::run(l, u, ns, all_short, static_cast<uint8_t*>(workspace), pieces, stream);
    return hipGetLastError() == hipSuccess ? THESEUS_WKV7_OK : THESEUS_WKV7_ERR_LAUNCH;
}

}  // extern "C"
