// Losses over a large vocabulary and their gradients without keeping the logits (C ABI:
// include/theseus_vocab.h, where the formulas are).
//
// Launches of one call, on the caller's stream:
//   targets        a teacher's: every token's q, Q, sum q log q and weight (a label's are made in rows)
//   sums           MEAN with several pieces: the sum of the weights (one workgroup, fixed order)
//   then for each piece of rows
//     logits       z's tiles on the matrix cores; of each tile (64 or 256 columns) a row's maximum and
//                  sum of exponentials are kept and, for gradients, the exponentials (float16,
//                  2^15 e^{z - tile maximum}: 11 significant bits down to e^-20 of the maximum);
//                  z at the targets is taken out of the accumulators
//     rows         log-sum-exp of a row from its tiles, the row's loss
//     sums         one piece: the reduced loss and, for MEAN, the sum of the weights; with gradients
//                  a workgroup of the next launch
//     probs        exponentials -> G in place (bfloat16: the one rounding of the gradients' left
//                  factor); at the target indices from their float32 z: p - 1 of a
//                  confident token would be lost in a rounded p
//     dhidden, dweight   G W and G^T H (vocab_gemm.h; float32 sums, rounded once)
//   sums           several pieces: the reduced loss
//
// The gradients take three products of 2 M V D operations, not the four of a backward that
// forms the logits again: with SUM and MEAN the upstream gradient is one number, applied to the
// results (theseus_vocab_scale); with NONE, up to THESEUS_VOCAB_MAX_KEPT bytes of exponentials are
// kept for the backward (1021 tokens of 50001 at width 2560: 990 -> 760 us), which otherwise makes them
// again (what that costs: beside the limit).
#include "../../include/theseus_vocab.h"
#include "../../include/theseus_wkv7.h"

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "vocab_gemm.h"

namespace vocab {

using wkv7::bf16_to_f32;
using wkv7::f32_to_bf16;
using wkv7::f32x2_to_bf16x2;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float E_SHIFT = 15.f;  // kept exponentials are 2^15 e^{z - max}
constexpr int SKIP = -1, BAD = -2;
constexpr int TWICE = 32;  // tokens

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }

__device__ __forceinline__ float wave_sum(float x) {
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}

// ---------------------------------------------------------------------------------- targets
struct Targets {
    long rows, vocab;
    int K, top_bf16;
    const int64_t* index;
    const void* top;
    const float* teacher_lse;
    const float* row_weight;
    float inv_T;
    int* j;        // [M][K] index, SKIP or BAD
    float* q;      // [M][K]
    float4* row;   // [M] {Q, sum q log q, weight, 0}
};

// labels: q = Q = 1
struct Labels {
    const int64_t* y;         // null: a teacher's targets
    const float* row_weight;
    long long ignore, vocab;
    __device__ __forceinline__ float4 row(long i) const {
        return make_float4(1.f, 0.f, y[i] == ignore ? 0.f : row_weight ? row_weight[i] : 1.f, 0.f);
    }
    __device__ __forceinline__ int place(long i) const {
        const int64_t v = y[i];
        return v == ignore ? SKIP : v < 0 || v >= vocab ? BAD : (int)v;
    }
};
// their weights ahead of the pieces; one thread a token
__global__ __launch_bounds__(256) void labels_kernel(Labels t, long rows, float4* row) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i < rows) row[i] = t.row(i);
}

// a teacher's logits: one wave a token
__global__ __launch_bounds__(256) void targets_kernel(Targets t) {
    constexpr int S = THESEUS_VOCAB_MAX_TOP / 64;
    const long i = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (i >= t.rows) return;
    const float weight = t.row_weight ? t.row_weight[i] : 1.f;
    float x[S], top = -INFINITY;
#pragma unroll
    for (int s = 0; s < S; s++) {
        const int k = 64 * s + lane;
        x[s] = -INFINITY;
        if (64 * s < t.K && k < t.K) {
            const long at = i * t.K + k;
            x[s] = (t.top_bf16 ? bf16_to_f32(static_cast<const uint16_t*>(t.top)[at]) : static_cast<const float*>(t.top)[at]) * t.inv_T;
        }
        top = fmaxf(top, x[s]);
    }
    float base;
    if (t.teacher_lse) {
        base = t.teacher_lse[i];
    } else {
        // (a token of whom the teacher kept nothing has q = 0 throughout)
        top = wave_max(top);
        float sum = 0.f;
#pragma unroll
        for (int s = 0; s < S; s++)
            if (64 * s < t.K) sum += x[s] == -INFINITY ? 0.f : expf(x[s] - top);
        base = top + logf(wave_sum(sum));
    }
    float Q = 0.f, H = 0.f;
#pragma unroll
    for (int s = 0; s < S; s++) {
        const int k = 64 * s + lane;
        if (k < t.K) {
            const float lq = x[s] - base, q = x[s] == -INFINITY ? 0.f : expf(lq);
            const long at = i * t.K + k;
            t.q[at] = q;
            const int64_t v = t.index[at];
            t.j[at] = q == 0.f ? SKIP : v < 0 || v >= t.vocab ? BAD : (int)v;
            Q += q;
            H += q == 0.f ? 0.f : q * lq;
        }
    }
    Q = wave_sum(Q);
    H = wave_sum(H);
    if (lane == 0) t.row[i] = make_float4(Q, H, weight, 0.f);
}

// MEAN: *inv = 1 / sum of the weights (0 where that is 0); with losses, *out = their sum, times
// *inv for MEAN.  One workgroup; 1024 partial sums, whatever its threads, added in a fixed order.
struct Sums {
    long rows;
    const float4* row;
    int mean;
    float* inv;
    const float* losses;
    float* out;
};
template <int THREADS> __device__ __forceinline__ void sums(const Sums& p) {
    __shared__ double red[2][16];
    const int t = threadIdx.x;
    for (int v = 0; v < 1024; v += THREADS) {
        double w = 0.0, s = 0.0;
#pragma unroll 4
        for (long i = v + t; i < p.rows; i += 1024) {
            if (p.mean) w += p.row[i].z;
            if (p.losses) s += p.losses[i];
        }
        for (int o = 32; o > 0; o >>= 1) {
            w += __shfl_xor(w, o, 64);
            s += __shfl_xor(s, o, 64);
        }
        if ((t & 63) == 0) red[0][(v + t) >> 6] = w, red[1][(v + t) >> 6] = s;
    }
    __syncthreads();
    if (t == 0) {
        double w = 0.0, s = 0.0;
        for (int k = 0; k < 16; k++) w += red[0][k], s += red[1][k];
        const double f = !p.mean ? 1.0 : w == 0.0 ? 0.0 : 1.0 / w;
        if (p.inv) *p.inv = (float)f;
        if (p.out) *p.out = (float)(s * f);
    }
}
__global__ __launch_bounds__(1024) void sums_kernel(Sums p) { sums<1024>(p); }

// a workgroup's tiles: every gridDim.x-th
template <class P> struct Places {
    const Tiles& t;
    int b = blockIdx.x;
    __device__ __forceinline__ explicit Places(const Tiles& tiles) : t(tiles) {}
    __device__ __forceinline__ Place place() const {
        const Where w = tile_of(t, b);
        const int s0 = w.part * t.steps;
        return Place{w.m * P::BM, w.n * P::BN, s0, min(t.steps, t.all - s0)};
    }
    __device__ __forceinline__ bool operator()(Place& p) {
        b += gridDim.x;
        if (b >= t.total) return false;
        p = place();
        return true;
    }
};

// ---------------------------------------------------------------------------------- logits
struct LogitsOut {
    int M, N, Ne;     // rows, vocabulary, columns kept (Ne >= N, zero beyond N)
    float scale;      // log2(e) / T
    float2* part;     // [M][tiles] {maximum of h . w, sum of 2^15 exp} of a tile
    int tiles;
    uint16_t* e;      // [..][lde]
    long lde;
    Labels labels;    // or
    const int* j;     // [M][K] targets
    float* z;         // [M][K] their h . w
    int K;
    int n0;           // the product's first column
};

// acc[tn][tm] of fragment code = tn TM + tm, the same for the whole wave (no indexed registers)
template <class P, int LO, int HI> __device__ __forceinline__ f32x4_t fragment(const P& g, int code) {
    if constexpr (HI - LO == 1) {
        f32x4_t a = g.acc[LO / P::TM][LO % P::TM];
        asm("" : "+v"(a));  // (a value here: joined as addresses, the accumulators would have to lie in memory)
        return a;
    }
    else if (code < (LO + HI) / 2) return fragment<P, LO, (LO + HI) / 2>(g, code);
    else return fragment<P, (LO + HI) / 2, HI>(g, code);
}
// h . w at the targets that lie in the workgroup's tile, out of the accumulators: the tile's tokens'
// targets are looked through (some thousand at a time), those in its columns listed in LDS, and each
// wave goes down the list for its own.  The list's order, which the atomics leave open, changes
// nothing.  (2048 x 131072 logits at D = 4096 and their gradient: 3412 us with 1 or 16 targets a token,
// 3497 with 64; dot products in a kernel of their own, D values of weight a target, 460 us for 32
// targets each of 8192 tokens, D = 5120.)
template <class P> __device__ __forceinline__ void pick_targets(const P& g, uint8_t* lds, const LogitsOut& o, int m0, int n0) {
    constexpr int READ = (P::EPILOGUE - 260) / (P::THREADS * 16), CHUNK = P::THREADS * 4 * READ;  // (fours a thread)
    uint32_t* list = reinterpret_cast<uint32_t*>(P::epilogue(lds));  // (64 entries are read at a time)
    int* count = reinterpret_cast<int*>(P::epilogue(lds) + CHUNK * 4 + 256);
    const int t = thread_here(), lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int total = min(P::BM, o.M - m0) * o.K, first = o.n0 + n0;
    const int* j = o.j + (long)m0 * o.K;
    for (int c0 = 0; c0 < total; c0 += CHUNK) {
        int4 v[READ];
        if (o.labels.y) {  // (one a token, at most 256)
#pragma unroll
            for (int r = 0; r < READ; r++) v[r] = make_int4(-1, -1, -1, -1);
            if (4 * t < total) {
                int x[4];
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = o.labels.place(m0 + min(4 * t + e, total - 1));
                v[0] = make_int4(x[0], x[1], x[2], x[3]);
            }
        } else {
#pragma unroll
            for (int r = 0; r < READ; r++) {  // (what a last four reads past the targets lies in the workspace)
                const int i = c0 + (r * P::THREADS + t) * 4;
                v[r] = i < total ? *reinterpret_cast<const int4*>(j + i) : make_int4(-1, -1, -1, -1);
            }
        }
        __syncthreads();
        if (t == 0) *count = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < READ; r++) {
            const int i = c0 + (r * P::THREADS + t) * 4, x[4] = {v[r].x, v[r].y, v[r].z, v[r].w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (i + e < total && (uint32_t)(x[e] - first) < (uint32_t)P::BN) {
                    const int m = (i + e) / o.K;
                    list[atomicAdd(count, 1)] = (uint32_t)m << 16 | (uint32_t)(x[e] - first) << 8 | (uint32_t)(i + e - m * o.K);
                }
        }
        __syncthreads();
        const int n = *count;
        for (int i = 0; i < n; i += 64) {
            const uint32_t own = list[i + lane];
            uint64_t mine = __ballot(i + lane < n && (int)(own >> 16) / (16 * P::TM) == wave / P::WN &&
                                     (int)((own >> 8) & 255) / (16 * P::TN) == wave % P::WN);
            for (; mine; mine &= mine - 1) {
                const uint32_t e = __builtin_amdgcn_readlane(own, __builtin_ctzll(mine));
                const int m = e >> 16, c = (e >> 8) & 255;
                const f32x4_t a = fragment<P, 0, P::TM * P::TN>(g, c / 16 % P::TN * P::TM + m / 16 % P::TM);
                const float z = (c & 2) ? (c & 1) ? a[3] : a[2] : (c & 1) ? a[1] : a[0];
                if ((lane & 15) == (m & 15) && lane >> 4 == ((c >> 2) & 3)) o.z[(long)(m0 + m) * o.K + (e & 255)] = z;
            }
        }
    }
    __syncthreads();
}

template <class P, bool KEEP> __device__ __forceinline__ void logits_done(P& g, uint8_t* lds, const LogitsOut& o, int m0, int n0) {
    pick_targets(g, lds, o, m0, n0);

    const int thread = thread_here(), lane = thread & 63, wave = thread >> 6, r16 = lane & 15, q = lane >> 4;
    const int wm = wave / P::WN, wn = wave % P::WN;
    const int mw = wm * P::TM * 16 + r16, nw = n0 + wn * P::TN * 16 + 4 * q;
    float* red = reinterpret_cast<float*>(P::epilogue(lds));  // [2][WN][BM]
    if (n0 + P::BN > o.N) {
#pragma unroll
        for (int tn = 0; tn < P::TN; tn++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (nw + 16 * tn + e >= o.N)
#pragma unroll
                    for (int tm = 0; tm < P::TM; tm++) g.acc[tn][tm][e] = -INFINITY;
    }
    float top[P::TM];
#pragma unroll
    for (int tm = 0; tm < P::TM; tm++) {
        top[tm] = g.acc[0][tm][0];
#pragma unroll
        for (int tn = 0; tn < P::TN; tn++)
#pragma unroll
            for (int e = 0; e < 4; e++) top[tm] = fmaxf(top[tm], g.acc[tn][tm][e]);
        top[tm] = fmaxf(top[tm], __shfl_xor(top[tm], 16, 64));
        top[tm] = fmaxf(top[tm], __shfl_xor(top[tm], 32, 64));
    }
    __syncthreads();
    if (q == 0)
#pragma unroll
        for (int tm = 0; tm < P::TM; tm++) red[wn * P::BM + mw + 16 * tm] = top[tm];
    __syncthreads();
#pragma unroll
    for (int tm = 0; tm < P::TM; tm++) {
        const int m = mw + 16 * tm;
        float all = red[m];
#pragma unroll
        for (int w = 1; w < P::WN; w++) all = fmaxf(all, red[w * P::BM + m]);
        float sum = 0.f;
#pragma unroll
        for (int tn = 0; tn < P::TN; tn++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x = exp2_(fmaf(g.acc[tn][tm][e] - all, o.scale, E_SHIFT));
                g.acc[tn][tm][e] = x;
                sum += x;
            }
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        top[tm] = all;
        if (q == 0) red[(P::WN + wn) * P::BM + m] = sum;
    }
    __syncthreads();
    if (wn == 0 && q == 0)
#pragma unroll
        for (int tm = 0; tm < P::TM; tm++) {
            const int m = mw + 16 * tm;
            if (m0 + m < o.M) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < P::WN; w++) sum += red[(P::WN + w) * P::BM + m];
                o.part[(long)(m0 + m) * o.tiles + n0 / P::BN] = make_float2(top[tm], sum);
            }
        }
    if constexpr (KEEP) {
        __syncthreads();
        store_rows<P>(lds, [&](int tn, int tm) {
            typedef _Float16 h4 __attribute__((ext_vector_type(4)));
            const f32x4_t a = g.acc[tn][tm];
            return __builtin_bit_cast(uint2, h4{(_Float16)a[0], (_Float16)a[1], (_Float16)a[2], (_Float16)a[3]});
        }, [&](int m, int n, uint4 v) {
            if (m0 + m < o.M && n0 + n < o.Ne) *reinterpret_cast<uint4*>(o.e + (long)(m0 + m) * o.lde + n0 + n) = v;
        });
    }
}

template <class P, bool KEEP>
__global__ __launch_bounds__(P::THREADS) void logits_kernel(Operand X, Operand Y, Tiles t, LogitsOut o) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[P::LDS];
    P g;
    g.template go<false>(lds, X, Y, Places<P>(t).place(), Places<P>(t), [&](const Place& at) { logits_done<P, KEEP>(g, lds, o, at.m0, at.n0); });
}

// ---------------------------------------------------------------------------------- rows
// One wave a token of the piece: maximum and sum over its tiles, the token's loss.  Nothing is
// taken from a rounded log-sum-exp, and products h . w are subtracted before they are scaled: for
// a confident token, lse - z and p - 1 are small differences of (z - maximum) and of the sum.
struct Rows {
    long rows;
    int tiles, K;
    const float2* part;
    Labels labels;  // their rows and places are written here
    float4* row;
    int* j;
    const float *q, *z;
    float T, scale;
    float2* norm;  // {maximum of h . w, 1 / sum of 2^15 exp}
    float* loss;
};
__global__ __launch_bounds__(256) void rows_kernel(Rows p) {
    const long i = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (i >= p.rows) return;
    const float2* part = p.part + i * p.tiles;
    float top = -INFINITY;
    for (int t = lane; t < p.tiles; t += 64) top = fmaxf(top, part[t].x);
    top = wave_max(top);
    float sum = 0.f;
    for (int t = lane; t < p.tiles; t += 64) sum += part[t].y * exp2_((part[t].x - top) * p.scale);
    sum = wave_sum(sum);
    const float lse = logf(sum * exp2_(-E_SHIFT));  // above the maximum
    const float4 row = p.labels.y ? p.labels.row(i) : p.row[i];
    float s = 0.f;
    for (int k = lane; k < p.K; k += 64) {
        const float q = p.q ? p.q[i * p.K + k] : 1.f;
        const int v = p.labels.y ? p.labels.place(i) : p.j[i * p.K + k];
        if (q != 0.f) s += v == BAD ? NAN : q * ((top - p.z[i * p.K + k]) * (LN2 * p.scale) + lse);
    }
    s = wave_sum(s);
    if (lane == 0) {
        if (p.labels.y) p.row[i] = row, p.j[i] = p.labels.place(i);
        p.norm[i] = make_float2(top, 1.f / sum);
        if (p.loss) p.loss[i] = row.z == 0.f ? 0.f : p.T * p.T * row.z * (s + row.y);
    }
}

// ---------------------------------------------------------------------------------- G
// G without its factor common to all tokens (T, and 1 / the sum of the weights for MEAN), which the
// products' epilogues apply in float32: with it, every label's -1 would become one and the same
// rounded number, an error of up to 2^-8 of the whole gradient.  For up to TWICE tokens, whose
// few large entries' roundings would not average out either (one token: the whole error of one
// number), G is kept as two rows of bfloat16, the rounded one and what rounding left: a step of
// the contraction over tokens has 64 rows anyway, and dhidden's smallest tile 64.
struct Probs {
    int M, K;               // the piece's tokens (its rows up to a multiple of 64 become zeros)
    int tiles;              // logits tiles of a row: main / cols of `cols` columns, then of `rest`
    int main, cols, rest;
    long lde;
    uint16_t* e;
    const float2* part;
    const float4* row;
    const float2* norm;
    const float* row_grad;
    const int* j;
    const float *q, *z;
    float scale;
    bool twice;             // rows 32 .. 63 take what rounding left of rows 0 .. 31
    bool sum;               // one row of workgroups more, whose first one makes `sums`
    Sums sums;
};
// blockIdx.x: PROBS columns of a row, 8 at a time a thread, then the targets among them; the rows
// backwards, from those that the logits wrote last to those that dhidden reads first.  (The sums are
// wanted by the products' epilogues only, and cost a launch of 4 us alone.)
constexpr int PROBS = 4096;
__global__ __launch_bounds__(256) void probs_kernel(Probs p) {
    __shared__ int js[THESEUS_VOCAB_MAX_TOP];
    __shared__ float qs[THESEUS_VOCAB_MAX_TOP];
    if (p.sum && blockIdx.y == 0) {
        if (blockIdx.x == 0) sums<256>(p.sums);
        return;
    }
    const long i = gridDim.y - 1 - blockIdx.y;
    const int t = threadIdx.x, n0 = blockIdx.x * PROBS;
    uint16_t *row = p.e + i * p.lde, *rest = row + 32 * p.lde;
    const float weight = i >= p.M ? 0.f : p.row[i].z;  // (0: whatever its upstream gradient, which may be infinite or NaN there)
    const float f = p.row_grad && weight != 0.f ? weight * p.row_grad[i] : weight;
    constexpr int G = PROBS / 2048;
    if (f == 0.f) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int n = n0 + (g * 256 + t) * 8;
            if (n < p.lde) {
                *reinterpret_cast<uint4*>(row + n) = make_uint4(0, 0, 0, 0);
                if (p.twice) *reinterpret_cast<uint4*>(rest + n) = make_uint4(0, 0, 0, 0);
            }
        }
        return;
    }
    uint4 u[G];
    float top[G];
#pragma unroll
    for (int g = 0; g < G; g++) {
        const int n = min(n0 + (g * 256 + t) * 8, (int)p.lde - 8);
        u[g] = *reinterpret_cast<const uint4*>(row + n);
        top[g] = p.part[i * p.tiles + (n < p.main ? n / p.cols : p.main / p.cols + (n - p.main) / p.rest)].x;
    }
    if (t < p.K) {
        js[t] = p.j[i * p.K + t];
        qs[t] = p.q ? p.q[i * p.K + t] : 1.f;
    }
    const float Q = p.row[i].x;
    const float2 norm = p.norm[i];
#pragma unroll
    for (int g = 0; g < G; g++) {
        const int n = n0 + (g * 256 + t) * 8;
        if (n >= p.lde) continue;
        const float c = f * Q * norm.y * exp2_((top[g] - norm.x) * p.scale);
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const uint32_t in[4] = {u[g].x, u[g].y, u[g].z, u[g].w};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const h2 h = __builtin_bit_cast(h2, in[e]);
            const float a = (float)h[0] * c, b = (float)h[1] * c;
            hi[e] = f32x2_to_bf16x2(a, b);
            lo[e] = f32x2_to_bf16x2(a - __uint_as_float(hi[e] << 16), b - __uint_as_float(hi[e] & 0xffff0000u));
        }
        *reinterpret_cast<uint4*>(row + n) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (p.twice) *reinterpret_cast<uint4*>(rest + n) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    __syncthreads();
    if (t < p.K) {  // (equal indices of one token write the same value)
        const int v = js[t];
        if (v >= n0 && v < n0 + PROBS) {
            float q = 0.f;
            for (int k = 0; k < p.K; k++) q += js[k] == v ? qs[k] : 0.f;
            const float g = f * (Q * (exp2_(fmaf(p.z[i * p.K + t] - norm.x, p.scale, E_SHIFT)) * norm.y) - q);
            row[v] = f32_to_bf16(g);
            if (p.twice) rest[v] = f32_to_bf16(g - bf16_to_f32(f32_to_bf16(g)));
        }
    }
}

// ---------------------------------------------------------------------------------- gradients
// bfloat16 C; float32 parts of the contraction; float32 sum over row pieces (bfloat16 from the last)
enum OutMode { OutBf16, OutPart, OutAdd };
struct GradOut {
    int M, N;
    uint16_t* c;   // [M][ldc]
    long ldc;
    float* f;      // OutPart: [splits][M][ldf]; OutAdd: [M][ldf]
    long ldf;
    int first, last;  // OutAdd: of the row pieces
    float T;              // the common factor T, times *inv where there is one
    const float* inv;
};

template <class P, OutMode MODE> __device__ __forceinline__ void grad_done(P& g, uint8_t* lds, const GradOut& o, int m0, int n0, int part) {
    const int thread = thread_here(), lane = thread & 63, wave = thread >> 6, r16 = lane & 15, q = lane >> 4;
    const int mw = m0 + (wave / P::WN) * P::TM * 16 + r16, nw = n0 + (wave % P::WN) * P::TN * 16 + 4 * q;
    if constexpr (MODE != OutBf16) {
#pragma unroll
        for (int tm = 0; tm < P::TM; tm++) {
            const long m = mw + 16 * tm;
#pragma unroll
            for (int tn = 0; tn < P::TN; tn++) {
                const int n = nw + 16 * tn;
                if (m >= o.M || n >= o.N) continue;
                if constexpr (MODE == OutPart) {
                    *reinterpret_cast<f32x4_t*>(o.f + ((long)part * o.M + m) * o.ldf + n) = g.acc[tn][tm];
                } else {
                    f32x4_t* f = reinterpret_cast<f32x4_t*>(o.f + m * o.ldf + n);
                    if (!o.first) g.acc[tn][tm] += *f;
                    if (!o.last) *f = g.acc[tn][tm];
                }
            }
        }
        if (MODE == OutPart || !o.last) return;
    }
    // (dweight is as large as the weight and not read again here: streamed past the caches it leaves them
    // to the weight and its own writing to the memory; 33 tokens, 56136 x 5120: the call 429 -> 374 us)
    const bool eight = (o.ldc & 7) == 0 && ((uintptr_t)o.c & 15) == 0;  // (N = ldc: eight columns are in or out together)
    const float f = o.inv ? o.T * *o.inv : o.T;
    store_rows<P>(lds, [&](int tn, int tm) {
        const f32x4_t a = g.acc[tn][tm] * f;
        return make_uint2(f32x2_to_bf16x2(a[0], a[1]), f32x2_to_bf16x2(a[2], a[3]));
    }, [&](int m, int n, uint4 v) {
        if (m0 + m >= o.M || n0 + n >= o.N) return;
        uint16_t* c = o.c + (long)(m0 + m) * o.ldc + n0 + n;
        if (eight) {
            typedef uint32_t u4 __attribute__((ext_vector_type(4)));
            if constexpr (P::LX == RowN) __builtin_nontemporal_store(__builtin_bit_cast(u4, v), reinterpret_cast<u4*>(c));
            else *reinterpret_cast<uint4*>(c) = v;
        } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            for (int e = 0; e < 8 && n0 + n + e < o.N; e++) c[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        }
    });
}
template <class P, OutMode MODE, bool SHORT = false>
__global__ __launch_bounds__(P::THREADS) void grad_kernel(Operand X, Operand Y, Tiles t, GradOut o) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[P::LDS];
    P g;
    g.template go<SHORT>(lds, X, Y, Places<P>(t).place(), Places<P>(t), [&](const Place& at) { grad_done<P, MODE>(g, lds, o, at.m0, at.n0, at.step0 / t.steps); });
}
// the parts of a contraction added in order, 4 columns a thread (twice = 32: and row m + 32's)
__global__ __launch_bounds__(256) void add_parts(GradOut o, int splits, int twice) {
    const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
    const long m = blockIdx.y;
    if (n >= o.N) return;
    f32x4_t a = {0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r <= twice; r += 32)  // (rows 32 .. 63: see above)
#pragma unroll 8
        for (int s = 0; s < splits; s++) a += *reinterpret_cast<const f32x4_t*>(o.f + ((long)s * o.M + m + r) * o.ldf + n);
    a *= o.inv ? o.T * *o.inv : o.T;
    for (int e = 0; e < 4 && n + e < o.N; e++) o.c[m * o.ldc + n + e] = f32_to_bf16(a[e]);
}

// copies rows of D elements (any alignment) to rows of Dp, zeros beyond D
__global__ __launch_bounds__(256) void pad_rows(long rows, int D, int Dp, const uint16_t* x, long ld, uint16_t* out) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= Dp) return;
    for (long i = blockIdx.y; i < rows; i += gridDim.y) out[i * Dp + c] = c < D ? x[i * ld + c] : 0;
}

// The gradients of a reduced loss, made with it for an upstream gradient of 1, times the one that came: each is
// rounded to bfloat16 twice then (2^-8 each, the second only where the factor is no power of two; 1 moves nothing).
// Float32 gradients from the forward to the backward would spare the first, at 4 bytes instead of 2 for each
// element of the weight.
__global__ __launch_bounds__(256) void scale_kernel(uint16_t* x, long nx, uint16_t* y, long ny, const float* factor) {
    const float f = *factor;
    if (f == 1.f) return;
    const long step = (long)gridDim.x * 256, first = (long)blockIdx.x * 256 + threadIdx.x;
    auto two = [&](uint32_t u) { return f32x2_to_bf16x2(__uint_as_float(u << 16) * f, __uint_as_float(u & 0xffff0000u) * f); };
    auto all = [&](uint16_t* v, long n) {
        const long n8 = ((uintptr_t)v & 15) == 0 ? n / 8 : 0;
        for (long i = first; i < n8; i += step) {
            uint4 u = reinterpret_cast<uint4*>(v)[i];
            u = make_uint4(two(u.x), two(u.y), two(u.z), two(u.w));
            reinterpret_cast<uint4*>(v)[i] = u;
        }
        for (long i = 8 * n8 + first; i < n; i += step) v[i] = f32_to_bf16(bf16_to_f32(v[i]) * f);
    };
    all(x, nx);
    all(y, ny);
}

__global__ __launch_bounds__(256) void zero_kernel(uint16_t* x, long n) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) x[i] = 0;
}

// ---------------------------------------------------------------------------------- host
// The tiles each product can be made in, and what they were measured to cost: us of a step of 64
// along the contraction and of the rest (first loads, epilogue) for as many tiles as run at
// once (per_cu on each CU).  From logits of 64 .. 1024 x 131072 at D = 1280 and 2560, dhidden of as
// many x 2560 from 131072, dweight of 131072 x 2560 from 64 .. 1024 tokens, and small ones.
// plan() takes the cheapest: e.g. 128 tokens' logits there take 152, 127, 176 and 234 us in the
// first four shapes, 512 tokens' 273, 346, 564 and 734, 384 tokens' 279 in tiles of 256 rows and 258 of
// 192; dhidden of 64 x 768 from 8192 31 us in 256 x 256 tiles (8 parts) and 13 in 64 x 64 (16), of
// 285 x 2048 from 101681 167 in 256 x 256 and 151 in 192 x 256 (16), of 100 x 5120 from 72799 198 in
// 128 x 128 one a CU and 168 two a CU.
struct Shape {
    int m, n, per_cu;
    double step, fixed;
};
using Logits0 = Product<256, 256, 4, 2, 2, RowK, RowK>;
using Logits1 = Product<128, 256, 2, 4, 3, RowK, RowK>;
using Logits2 = Product<64, 256, 1, 8, 4, RowK, RowK>;
using Logits3 = Product<64, 64, 2, 4, 4, RowK, RowK>;
using Logits4 = Product<192, 256, 4, 2, 2, RowK, RowK>;
constexpr Shape LOGITS[] = {{256, 256, 1, 1.5, 7}, {128, 256, 1, .95, 5}, {64, 256, 1, .78, 4}, {64, 64, 2, .5, 2.3}, {192, 256, 1, 1.27, 5.5}};
using Dhidden0 = Product<256, 256, 4, 2, 2, RowK, RowN>;
using Dhidden1 = Product<128, 128, 2, 4, 2, RowK, RowN>;
using Dhidden2 = Product<64, 256, 1, 8, 4, RowK, RowN>;
using Dhidden3 = Product<64, 64, 2, 4, 4, RowK, RowN>;
using Dhidden5 = Product<192, 256, 4, 2, 2, RowK, RowN>;
constexpr Shape DHIDDEN[] = {{256, 256, 1, 1.75, 12}, {128, 128, 1, .8, 5}, {64, 256, 1, .85, 8}, {64, 64, 1, .45, 3}, {128, 128, 2, 1.45, 7}, {192, 256, 1, 1.5, 8.5}};
using Dweight0 = Product<256, 256, 4, 2, 2, RowN, RowN>;
using Dweight1 = Product<128, 128, 2, 4, 2, RowN, RowN>;
constexpr Shape DWEIGHT[] = {{256, 256, 1, 1.62, 6.7}, {128, 128, 2, 1.03, 4.1}};
constexpr double LAUNCH = 3, BYTES = 5e6;  // us of one more launch; bytes a us
constexpr int TOGETHER = 1024;             // rows of a product whose tiles run together (see tiles())

static long up(long x, long to) { return (x + to - 1) / to * to; }
static long ceil_div(long x, long y) { return (x + y - 1) / y; }

struct Plan {
    long M, V, D, K, Dp, lde, piece;  // Dp: width in the products; lde: kept columns; piece: rows
    int pieces, tiles;                // row pieces; logits tiles of a row
    bool grads, padh, padw, twice;    // padh, padw: hidden, weight copied to rows of Dp
    int logits, rest, dhidden, dweight, wrest;  // indices into the shapes
    long main;                        // columns of the vocabulary in shape `logits`, the others in `rest`
    long wmain;                       // rows of dweight in shape `dweight`, the others in `wrest`
    int splits;                       // of dhidden's contraction
    size_t j, q, row, z, part, norm, loss, inv, e, kept, acc, parts, hidden, weight, bytes;
};

constexpr long MAX_PIECE = 32768;  // rows: a grid's y dimension
// Elements from row to row in the products, which address a tile's rows by 32-bit byte offsets.  Hidden
// states further apart (the last token of each of several long sequences) are copied, a weight is refused.
constexpr long MAX_STRIDE = 1l << 21;

static int device_cus() {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 256;
    return n > 0 ? n : 256;
}

static int check(const theseus_vocab_loss_args* a) {
    if (!a) return THESEUS_WKV7_ERR_NULL;
    if (a->rows < 0 || a->rows > (1ll << 30) || a->vocab < 1 || a->vocab > (1ll << 22) || a->width < 1 || a->width > (1 << 17) ||
        a->targets < 1 || a->targets > THESEUS_VOCAB_MAX_TOP || (!a->top_values && a->targets != 1) || a->hidden_stride < a->width ||
        a->weight_stride < a->width || a->piece_rows < 0 || !(a->temperature > 0.f) || !isfinite(a->temperature))
        return THESEUS_WKV7_ERR_SHAPE;
    if (a->vocab > 1 && a->weight_stride > MAX_STRIDE) return THESEUS_WKV7_ERR_SHAPE;
    if (a->top_dtype != THESEUS_VOCAB_BF16 && a->top_dtype != THESEUS_VOCAB_FP32) return THESEUS_WKV7_ERR_DTYPE;
    if (a->reduction < THESEUS_VOCAB_NONE || a->reduction > THESEUS_VOCAB_MEAN || a->phase < THESEUS_VOCAB_ALL ||
        a->phase > THESEUS_VOCAB_GRADIENTS || (a->phase != THESEUS_VOCAB_ALL && a->reduction != THESEUS_VOCAB_NONE))
        return THESEUS_WKV7_ERR_FLAGS;
    return THESEUS_WKV7_OK;
}

// us of a product of M x N outputs: its full rounds of tiles and a last one with fewer, each the
// tiles' own time or the reading of the weight behind them (`bytes` in all, once for TOGETHER
// rows), whichever is longer, and a little of the other.  A last round's tiles run faster, the fewer
// the more (the clock; 3088 tokens' dweight of 25163 x 2048, 24 tiles of 256: 44 us for 86)
static double both(double a, double b) { return a > b ? a + .1 * b : b + .1 * a; }
static double cost(const Shape& c, long M, long N, long steps, double bytes, int cus) {
    const long t = ceil_div(M, c.m) * ceil_div(N, c.n), slots = (long)cus * c.per_cu, full = t / slots, left = t % slots;
    const double tile = c.fixed + (double)steps * c.step, read = ceil_div(M, TOGETHER) * bytes / BYTES / t;
    return (full ? full * both(tile, slots * read) : 0) + (left ? both(full ? tile * (.6 + .4 * left / slots) : tile, left * read) : 0);
}
template <int N> static int best(const Shape (&c)[N], long M, long cols, long steps, double bytes, int cus, double* us) {
    int b = 0;
    double u = 0;
    for (int i = 0; i < N; i++) {
        const double x = cost(c[i], M, cols, steps, bytes, cus);
        if (i == 0 || x < u) b = i, u = x;
    }
    *us = u;
    return b;
}

static Plan plan(const theseus_vocab_loss_args* a) {
    Plan p{};
    p.M = a->rows, p.V = a->vocab, p.D = a->width, p.K = a->targets;
    p.Dp = up(p.D, BK);
    // (the products read rows of whole steps, 16 bytes at a time; the stride of one row is not used)
    auto pad = [&](const void* x, long rows, long stride) {
        return p.D != p.Dp || (uintptr_t)x % 16 || (rows > 1 && (stride % 8 || stride > MAX_STRIDE));
    };
    p.padh = pad(a->hidden, p.M, a->hidden_stride), p.padw = pad(a->weight, p.V, a->weight_stride);
    p.grads = a->dhidden || a->dweight || a->phase != THESEUS_VOCAB_ALL;
    p.lde = up(p.V, BK);
    long cap = a->piece_rows ? up(a->piece_rows < MAX_PIECE ? a->piece_rows : MAX_PIECE, 256) : p.grads ? (2l << 30) / (2 * p.lde) / 256 * 256 : MAX_PIECE;
    cap = cap < 256 ? 256 : cap > MAX_PIECE ? MAX_PIECE : cap;
    p.pieces = (int)ceil_div(p.M, cap);
    p.piece = up(ceil_div(p.M, p.pieces ? p.pieces : 1), 256);
    p.pieces = (int)ceil_div(p.M, p.piece ? p.piece : 256);
    const long rows = p.M == 0 ? 1 : p.M < p.piece ? p.M : p.piece;  // of the largest piece (no tokens: nothing is launched for them)
    p.twice = p.M <= TWICE;
    const int cus = device_cus();
    const long steps = p.Dp / BK;
    // one shape for all columns, or full rounds of one and the remaining columns in another
    // (1021 x 50001 at D = 2560: 784 tiles of 256 x 256, 3.06 rounds of 256 CUs; 296 -> 241 us)
    double us, least;
    const double column = (double)p.Dp * 2;
    p.logits = p.rest = best(LOGITS, rows, p.V, steps, p.V * column, cus, &least);
    p.main = p.V;
    for (int i = 0; i < (int)(sizeof LOGITS / sizeof *LOGITS); i++) {
        const Shape& c = LOGITS[i];
        const long tm = ceil_div(rows, c.m), slots = (long)cus * c.per_cu, n = tm * ceil_div(p.V, c.n) / slots * slots / tm * c.n;
        if (n <= 0 || n >= p.V) continue;
        const int r = best(LOGITS, rows, p.V - n, steps, (p.V - n) * column, cus, &us);
        us += cost(c, rows, n, steps, n * column, cus) + LAUNCH;
        if (us < least) least = us, p.logits = i, p.main = n, p.rest = r;
    }
    p.tiles = (int)(ceil_div(p.main, LOGITS[p.logits].n) + ceil_div(p.V - p.main, LOGITS[p.rest].n));
    if (a->dhidden) {
        // its contraction, the vocabulary, is long and its tiles few: float32 parts that fill the
        // CUs, added afterwards
        const long all = p.lde / BK, gm = p.twice ? 64 : rows;
        const double read = (double)ceil_div(gm, TOGETHER) * p.V * column / BYTES;
        least = 0;
        for (int i = 0; i < (int)(sizeof DHIDDEN / sizeof *DHIDDEN); i++) {
            const Shape& c = DHIDDEN[i];
            const long t = ceil_div(gm, c.m) * ceil_div(p.D, c.n);
            const long slots = (long)cus * c.per_cu;
            for (int r = 1; r <= 12; r++) {  // few parts, or as many as fit 1 .. 4 rounds (every call comes by here: few candidates)
                const long s = r <= 8 ? r : (r - 8) * slots / t;
                if (s > all || s > 64 || (r > 8 && s <= 8)) continue;
                us = both(ceil_div(t * s, slots) * (c.fixed + ceil_div(all, s) * c.step), read) +
                     (s > 1 ? LAUNCH + (double)s * gm * p.D * 8 / BYTES : 0);
                if (least == 0 || us < least) least = us, p.dhidden = i, p.splits = (int)s;
            }
        }
    }
    if (a->dweight) {
        const long k = ceil_div(rows, BK);
        p.dweight = p.wrest = best(DWEIGHT, p.V, p.D, k, 0, cus, &least);
        p.wmain = p.V;
        // (as the logits' columns; 2604 tokens, 53714 x 768: 2.46 rounds of 256 x 256 tiles, 207 -> 195 us;
        // the smaller tiles are slower in full rounds)
        const Shape& c = DWEIGHT[0];
        const long tn = ceil_div(p.D, c.n), m = ceil_div(p.V, c.m) * tn / cus * cus / tn * c.m;
        if (m > 0 && m < p.V) {
            const int r = best(DWEIGHT, p.V - m, p.D, k, 0, cus, &us);
            us += cost(c, m, p.D, k, 0, cus) + LAUNCH;
            if (us < least) p.dweight = 0, p.wmain = m, p.wrest = r;
        }
    }
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) / 256 * 256;
        return here;
    };
    p.j = take(p.M * p.K * 4);
    p.q = take(a->top_values ? p.M * p.K * 4 : 0);
    p.row = take(p.M * 16);
    p.z = take(p.M * p.K * 4);
    p.loss = take(a->loss && a->reduction != THESEUS_VOCAB_NONE ? p.M * 4 : 0);
    p.inv = take(4);
    p.norm = take(rows * 8);
    p.part = take((size_t)rows * p.tiles * 8);
    p.e = take(p.grads ? (size_t)up(rows, BK) * p.lde * 2 : 0);
    p.kept = at;
    if (a->phase != THESEUS_VOCAB_ALL) at = 0;  // (what is above lies in a->kept)
    p.acc = take(a->dweight && p.pieces > 1 ? (size_t)p.V * up(p.D, 4) * 4 : 0);
    p.parts = take(p.splits > 1 || p.twice ? (size_t)p.splits * (p.twice ? 64 : rows) * up(p.D, 4) * 4 : 0);
    p.hidden = take(p.padh ? (size_t)p.M * p.Dp * 2 : 0);
    p.weight = take(p.padw ? (size_t)p.V * p.Dp * 2 : 0);
    p.bytes = at;
    if (a->phase == THESEUS_VOCAB_FORWARD && !p.padh && !p.padw) p.bytes = 0;
    return p;
}

static Tiles tiles(long M, long N, int BM, int BN, long K, int splits) {
    Tiles t;
    t.m = (int)ceil_div(M, BM), t.n = (int)ceil_div(N, BN);
    t.all = (int)(K / BK);
    t.steps = (int)ceil_div(t.all, splits);
    t.splits = (int)ceil_div(t.all, t.steps);
    t.total = t.m * t.n * t.splits;
    // m tiles that run together, 1024 rows: with 256 x 256 tiles and 8192 rows 4 tiles took 4.46 ms for
    // dweight, 8 4.63 and 2 4.51; smaller tiles of few rows would read the other operand again
    const int group = TOGETHER / BM;
    t.group = t.m < group ? t.m : group;
    return t;
}

// workgroups of a product: as many as run at once, each with its tiles, or (few steps, and not go()'s
// SHORT form) one a tile
template <class P> static unsigned groups(const Tiles& t, int cus, bool few = false) {
    const int slots = cus * (163840 / P::LDS < 2 ? 1 : 2) / 8 * 8;
    return P::KEPT && (few || t.all - (t.splits - 1) * t.steps > P::NST) && slots > 0 && t.total > slots ? slots : t.total;
}

static int run(const theseus_vocab_loss_args* a, const Plan& p, uint8_t* ws, hipStream_t st) {
    const int cus = device_cus();
    uint8_t* first = a->phase != THESEUS_VOCAB_ALL ? static_cast<uint8_t*>(a->kept) : ws;
    auto at = [&](size_t off) { return first + off; };
    const bool forward = a->phase != THESEUS_VOCAB_GRADIENTS, gradients = p.grads && a->phase != THESEUS_VOCAB_FORWARD;
    int* j = reinterpret_cast<int*>(at(p.j));
    float* q = a->top_values ? reinterpret_cast<float*>(at(p.q)) : nullptr;
    float4* row = reinterpret_cast<float4*>(at(p.row));
    float* z = reinterpret_cast<float*>(at(p.z));
    float* inv = a->reduction == THESEUS_VOCAB_MEAN ? reinterpret_cast<float*>(at(p.inv)) : nullptr;
    float2* norm = reinterpret_cast<float2*>(at(p.norm));
    float2* part = reinterpret_cast<float2*>(at(p.part));
    uint16_t* e = reinterpret_cast<uint16_t*>(at(p.e));
    const bool reduce = a->loss && a->reduction != THESEUS_VOCAB_NONE;
    float* losses = reduce ? reinterpret_cast<float*>(at(p.loss)) : a->loss;
    const uint16_t* H = static_cast<const uint16_t*>(a->hidden);
    const uint16_t* W = static_cast<const uint16_t*>(a->weight);
    long ldh = p.M == 1 ? p.Dp : a->hidden_stride, ldw = p.V == 1 ? p.Dp : a->weight_stride;
    const float inv_T = 1.f / a->temperature;
    if (p.M == 0) {
        if (reduce) sums_kernel<<<1, 1024, 0, st>>>(Sums{0, nullptr, 0, nullptr, nullptr, a->loss});
        if (a->dweight) zero_kernel<<<1024, 256, 0, st>>>(static_cast<uint16_t*>(a->dweight), p.V * p.D);
        return 0;
    }
    auto padded = [&](const uint16_t* x, long rows, long& ld, size_t to) {
        uint16_t* out = reinterpret_cast<uint16_t*>(ws + to);
        pad_rows<<<dim3((unsigned)ceil_div(p.Dp, 256), (unsigned)(rows < 32768 ? rows : 32768)), 256, 0, st>>>(rows, (int)p.D, (int)p.Dp, x, ld, out);
        ld = p.Dp;
        return static_cast<const uint16_t*>(out);
    };
    if (p.padh) H = padded(H, p.M, ldh, p.hidden);
    if (p.padw) W = padded(W, p.V, ldw, p.weight);
    if (forward && a->top_values) {
        // (a launch has fewer than 2^32 threads, 64 a token)
        const long most = 1l << 25, size = a->top_dtype == THESEUS_VOCAB_BF16 ? 2 : 4;
        for (long i = 0; i < p.M; i += most) {
            const long n = p.M - i < most ? p.M - i : most;
            const Targets t{n, p.V, (int)p.K, a->top_dtype == THESEUS_VOCAB_BF16, a->index + i * p.K, static_cast<const uint8_t*>(a->top_values) + i * p.K * size,
                            a->teacher_lse ? a->teacher_lse + i : nullptr, a->row_weight ? a->row_weight + i : nullptr, inv_T, j + i * p.K, q + i * p.K, row + i};
            targets_kernel<<<(unsigned)ceil_div(n, 4), 256, 0, st>>>(t);
        }
    }
    auto labels = [&](long i0) {
        return Labels{a->top_values ? nullptr : a->index + i0, a->row_weight ? a->row_weight + i0 : nullptr, a->ignore_index, p.V};
    };
    const bool mean = inv != nullptr;
    auto sums_of = [&](float* to, const float* from, float* out) { return Sums{p.M, row, mean, to, from, out}; };
    if (mean && p.grads && p.pieces > 1) {
        if (!a->top_values) labels_kernel<<<(unsigned)ceil_div(p.M, 256), 256, 0, st>>>(labels(0), p.M, row);
        sums_kernel<<<1, 1024, 0, st>>>(sums_of(inv, nullptr, nullptr));
    }

    for (int piece = 0; piece < p.pieces; piece++) {
        const long i0 = piece * p.piece, m = p.M - i0 < p.piece ? p.M - i0 : p.piece;
        const uint16_t* Hp = H + i0 * ldh;
        auto logits = [&](int shape, long n0, long n1, int tile0) {
            const Operand X{Hp, ldh, (int)m, (int)p.Dp}, Y{W + n0 * ldw, ldw, (int)(n1 - n0), (int)p.Dp};
            const LogitsOut lo{(int)m, (int)(n1 - n0), (int)((n1 == p.V ? p.lde : n1) - n0), LOG2E * inv_T, part + tile0, p.tiles,
                               p.grads ? e + n0 : nullptr, p.lde, labels(i0), j + i0 * p.K, z + i0 * p.K, (int)p.K, (int)n0};
            auto launch = [&](auto tag) {
                using P = decltype(tag);
                const Tiles tl = tiles(m, n1 - n0, P::BM, P::BN, p.Dp, 1);
                if (p.grads) logits_kernel<P, true><<<groups<P>(tl, cus), P::THREADS, 0, st>>>(X, Y, tl, lo);
                else logits_kernel<P, false><<<groups<P>(tl, cus), P::THREADS, 0, st>>>(X, Y, tl, lo);
            };
            switch (shape) {
                case 0: launch(Logits0{}); break;
                case 1: launch(Logits1{}); break;
                case 2: launch(Logits2{}); break;
                case 4: launch(Logits4{}); break;
                default: launch(Logits3{});
            }
        };
        if (forward) {
            logits(p.logits, 0, p.main, 0);
            if (p.main < p.V) logits(p.rest, p.main, p.V, (int)ceil_div(p.main, LOGITS[p.logits].n));
        }
        const Rows rw{m, p.tiles, (int)p.K, part, labels(i0), row + i0, j + i0 * p.K, q ? q + i0 * p.K : nullptr, z + i0 * p.K,
                      a->temperature, LOG2E * inv_T, norm, losses ? losses + i0 : nullptr};
        if (forward) rows_kernel<<<(unsigned)ceil_div(m, 4), 256, 0, st>>>(rw);
        const bool sum = p.pieces == 1 && (reduce || (mean && p.grads));
        const Sums su = sums_of(inv, reduce ? losses : nullptr, reduce ? a->loss : nullptr);
        if (sum && !gradients) sums_kernel<<<1, 1024, 0, st>>>(su);
        if (!gradients) continue;

        const long mp = up(m, BK);
        const Probs pr{(int)m, (int)p.K, p.tiles, (int)(p.main < p.V ? p.main : p.lde), LOGITS[p.logits].n, LOGITS[p.rest].n, p.lde, e, part, row + i0, norm,
                       a->row_grad ? a->row_grad + i0 : nullptr, j + i0 * p.K, q ? q + i0 * p.K : nullptr, z + i0 * p.K, LOG2E * inv_T, p.twice, sum, su};
        probs_kernel<<<dim3((unsigned)ceil_div(p.lde, PROBS), (unsigned)((p.twice ? 32 : mp) + sum)), 256, 0, st>>>(pr);
        if (a->dhidden) {
            uint16_t* dh = static_cast<uint16_t*>(a->dhidden) + i0 * p.D;
            const long gm = p.twice ? 64 : m;  // rows of G
            const Operand GX{e, p.lde, (int)gm, (int)p.lde}, WY{W, ldw, (int)p.Dp, (int)p.V};
            float* parts = reinterpret_cast<float*>((ws + p.parts));
            const GradOut go{(int)gm, (int)p.D, dh, p.D, parts, up(p.D, 4), 0, 0, a->temperature, inv};
            auto dhidden = [&](auto tag) {
                using P = decltype(tag);
                const Tiles tl = tiles(gm, p.D, P::BM, P::BN, p.lde, p.splits);
                if (tl.splits > 1 || p.twice) {
                    grad_kernel<P, OutPart><<<groups<P>(tl, cus), 512, 0, st>>>(GX, WY, tl, go);
                    add_parts<<<dim3((unsigned)ceil_div(p.D, 1024), (unsigned)m), 256, 0, st>>>(go, tl.splits, p.twice ? 32 : 0);
                } else {
                    grad_kernel<P, OutBf16><<<groups<P>(tl, cus), 512, 0, st>>>(GX, WY, tl, go);
                }
            };
            switch (p.dhidden) {
                case 0: dhidden(Dhidden0{}); break;
                case 1: case 4: dhidden(Dhidden1{}); break;
                case 2: dhidden(Dhidden2{}); break;
                case 5: dhidden(Dhidden5{}); break;
                default: dhidden(Dhidden3{});
            }
        }
        if (a->dweight) {
            const Operand HY{Hp, ldh, (int)p.Dp, (int)m, p.twice};
            auto dweight = [&](auto tag, long v0, long v1) {
                using P = decltype(tag);
                const Operand GX{e + v0, p.lde, (int)((v1 == p.V ? p.lde : v1) - v0), (int)mp};
                const GradOut go{(int)(v1 - v0), (int)p.D, static_cast<uint16_t*>(a->dweight) + v0 * p.D, p.D,
                                 reinterpret_cast<float*>((ws + p.acc)) + v0 * up(p.D, 4), up(p.D, 4), piece == 0, piece == p.pieces - 1,
                                 a->temperature, inv};
                const Tiles tl = tiles(v1 - v0, p.D, P::BM, P::BN, mp, 1);
                const bool few = tl.all <= P::NST;  // up to 128 tokens
                if (p.pieces > 1) grad_kernel<P, OutAdd><<<groups<P>(tl, cus), 512, 0, st>>>(GX, HY, tl, go);
                else if (few) grad_kernel<P, OutBf16, true><<<groups<P>(tl, cus, true), 512, 0, st>>>(GX, HY, tl, go);
                else grad_kernel<P, OutBf16><<<groups<P>(tl, cus), 512, 0, st>>>(GX, HY, tl, go);
            };
            if (p.dweight == 0) dweight(Dweight0{}, 0, p.wmain);
            else dweight(Dweight1{}, 0, p.wmain);
            if (p.wmain < p.V) {
                if (p.wrest == 0) dweight(Dweight0{}, p.wmain, p.V);
                else dweight(Dweight1{}, p.wmain, p.V);
            }
        }
    }
    if (reduce && p.pieces > 1) sums_kernel<<<1, 1024, 0, st>>>(sums_of(inv, losses, a->loss));
    return 0;
}

}  // namespace vocab

extern "C" {

size_t theseus_vocab_loss_workspace_size(const theseus_vocab_loss_args* args) {
    return vocab::check(args) ? 0 : vocab::plan(args).bytes;
}

size_t theseus_vocab_loss_kept_size(const theseus_vocab_loss_args* args) {
    if (vocab::check(args) || !args->rows || args->reduction != THESEUS_VOCAB_NONE) return 0;
    theseus_vocab_loss_args a = *args;
    a.phase = THESEUS_VOCAB_FORWARD;
    const vocab::Plan p = vocab::plan(&a);
    return p.pieces == 1 && p.kept <= (size_t)THESEUS_VOCAB_MAX_KEPT ? p.kept : 0;
}

int theseus_vocab_loss(const theseus_vocab_loss_args* a, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (int e = vocab::check(a)) return e;
    if (a->rows && (!a->hidden || !a->weight || !a->index)) return THESEUS_WKV7_ERR_NULL;
    if (a->phase != THESEUS_VOCAB_ALL) {
        if (!theseus_vocab_loss_kept_size(a)) return THESEUS_WKV7_ERR_SHAPE;
        if (!a->kept) return THESEUS_WKV7_ERR_NULL;
    }
    const vocab::Plan p = vocab::plan(a);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes)) return THESEUS_WKV7_ERR_WORKSPACE;
    vocab::run(a, p, static_cast<uint8_t*>(workspace), stream);
    return hipGetLastError() == hipSuccess ? THESEUS_WKV7_OK : THESEUS_WKV7_ERR_LAUNCH;
}

int theseus_vocab_scale(void* x, long long nx, void* y, long long ny, const float* factor, hipStream_t stream) {
    if (nx < 0 || ny < 0) return THESEUS_WKV7_ERR_SHAPE;
    if ((nx && !x) || (ny && !y) || !factor) return THESEUS_WKV7_ERR_NULL;
    if (!nx && !ny) return THESEUS_WKV7_OK;
    const long blocks = vocab::ceil_div(nx > ny ? nx : ny, 8 * 256);
    vocab::scale_kernel<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, stream>>>(static_cast<uint16_t*>(x), nx,
                                                                                       static_cast<uint16_t*>(y), ny, factor);
    return hipGetLastError() == hipSuccess ? THESEUS_WKV7_OK : THESEUS_WKV7_ERR_LAUNCH;
}

}  // extern "C"
