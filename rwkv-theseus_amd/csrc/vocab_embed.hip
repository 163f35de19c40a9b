// Token embedding and its gradient (C ABI: include/theseus_embed.h), gfx950.
//
//   lookup   out_i = scale weight_{ids_i}: a gather, bound by the rows read and written.
//   grad     dweight_v = scale sum over the tokens i of v, in their order, of grad_i.
//
// The gradient sorts the tokens by index (stable, so that each index' tokens keep their order),
// cuts the sorted list into runs of `each` tokens and sums every run's stretches of one index in
// registers, no atomics.  A stretch inside one run is a finished row; one that crosses runs leaves a
// float32 part in each, which a last launch adds in order: a token that fills half of a batch (a
// space, a padding) costs no more than the others.  Three launches up to ONE tokens:
//   sort_fill    workgroup 0 sorts in LDS, least significant digit first; the others meanwhile
//                write the table's zeros, most of the bytes: rows with tokens are written again.
//   sum_runs     a run of tokens x 256 threads of eight columns, 16 tokens' rows in flight (8 of float32).
//   add_parts    where a stretch begins that crosses runs: its parts in order.
// More tokens are sorted by many workgroups: digit counts, their prefix sums, places, per digit.
// Few tokens (up to 1024 of narrow rows, 256 of wide ones) take one launch, few_tokens.
#include "../../include/theseus_embed.h"
#include "../../include/theseus_wkv7.h"

#include <type_traits>

#include "wkv7_common.h"

namespace embed {

using wkv7::bf16_to_f32;
using wkv7::f32x2_to_bf16x2;
using wkv7::f32_to_bf16;

static long ceil_div(long x, long y) { return (x + y - 1) / y; }

// N values of a row at an address aligned to its elements only (the hardware loads and stores
// whole vectors at any address; odd widths have no other rows)
template <int N, typename T> struct Vec {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T> struct Vec<1, T> {
    typedef T type;
};
// ONCE: values that nobody reads again, past the caches
template <int N, bool ONCE = false, typename T> __device__ __forceinline__ void load(float (&x)[N], const T* p) {
    const auto* at = reinterpret_cast<const typename Vec<N, T>::type*>(p);
    const auto v = ONCE ? __builtin_nontemporal_load(at) : *at;
    auto value = [](auto y) {
        if constexpr (sizeof(T) == 2) return bf16_to_f32(y);
        else return y;
    };
    if constexpr (N == 1) x[0] = value(v);
    else
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = value(v[e]);
}
template <int N> __device__ __forceinline__ void store(uint16_t* p, const float (&x)[N]) {
    if constexpr (N == 1) *p = f32_to_bf16(x[0]);
    else {
        typedef uint32_t words __attribute__((ext_vector_type(N / 2), aligned(2)));
        words v;
#pragma unroll
        for (int e = 0; e < N / 2; e++) v[e] = f32x2_to_bf16x2(x[2 * e], x[2 * e + 1]);
        *reinterpret_cast<words*>(p) = v;
    }
}
template <int N> __device__ __forceinline__ void store(float* p, const float (&x)[N]) {
    if constexpr (N == 1) *p = x[0];
    else {
        typename Vec<N, float>::type v;
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = x[e];
        *reinterpret_cast<typename Vec<N, float>::type*>(p) = v;
    }
}

// A row is worked on in chunks of N columns (N = 8, or 1 where D < 8); the last one lies at the
// row's end and may overlap the one before it, whose values it makes again.
template <int N> __device__ __forceinline__ int column(int chunk, int D) { return min(chunk * N, D - N); }

// ------------------------------------------------------------------------------ lookup
// EACH chunks a thread, their loads in flight together; chunks behind the last one are the last one.
template <int N, int EACH, typename W, typename O>
__global__ __launch_bounds__(256) void lookup(long M, long V, int D, const int64_t* __restrict__ ids, const W* __restrict__ w,
                                              long ldw, float scale, O* __restrict__ out) {
    const unsigned per = (D + N - 1) / N;
    const long blocks = (M * per + 256 * EACH - 1) / (256 * EACH);
    for (long b = blockIdx.x; b < blocks; b += gridDim.x) {
        const long start = b * (256 * EACH), row0 = start / per;
        const unsigned off = (unsigned)(start - row0 * per) + threadIdx.x;
        long row[EACH], id[EACH];
        int col[EACH];
#pragma unroll
        for (int u = 0; u < EACH; u++) {
            const unsigned c = off + 256 * u, r = c / per;
            row[u] = min(row0 + r, M - 1);
            col[u] = column<N>(c - r * per, D);
            id[u] = ids[row[u]];
        }
        float x[EACH][N];
#pragma unroll
        for (int u = 0; u < EACH; u++) load<N>(x[u], w + ((uint64_t)id[u] < (uint64_t)V ? id[u] : 0) * ldw + col[u]);
#pragma unroll
        for (int u = 0; u < EACH; u++) {
            const float s = (uint64_t)id[u] < (uint64_t)V ? scale : __builtin_nanf("");
#pragma unroll
            for (int e = 0; e < N; e++) x[u][e] *= s;
            store<N>(out + row[u] * D + col[u], x[u]);
        }
    }
}

// ------------------------------------------------------------------------------ sort
constexpr int ONE = 16384;    // tokens that one workgroup sorts
constexpr int THREADS = 1024; // of a sorting workgroup: 16 waves, each with consecutive tokens
constexpr int WAVES = THREADS / 64;
constexpr int MAX_BITS = 10;  // of a digit
constexpr int BLOCK = 4096;   // tokens of a workgroup where there are more

// What a token is sorted by: its index, V for those that add nothing.
__device__ __forceinline__ uint32_t key_of(int64_t id, int64_t V, int64_t skip) {
    return (uint64_t)id < (uint64_t)V && id != skip ? (uint32_t)id : (uint32_t)V;
}

struct Digits {
    int bits, passes;
};
static Digits digits(long V) {  // of 0 .. V
    int n = 1;
    while (V >> n) n++;
    const int passes = (n + MAX_BITS - 1) / MAX_BITS;
    return {(n + passes - 1) / passes, passes};
}

__device__ __forceinline__ uint32_t digit_of(uint32_t key, int shift, int bits) { return key >> shift & ((1u << bits) - 1); }

// For this workgroup's values, wave after wave and ROUNDS x 64 a wave: each value's place among
// those of its digit, in order (`rank`: within its wave; count[wave][digit]: of the waves before).
// all[digit] is the workgroup's count.
template <int ROUNDS>
__device__ __forceinline__ void rank_digits(const uint32_t (&key)[ROUNDS], uint32_t (&rank)[ROUNDS], int shift, int bits, uint16_t* count,
                                            uint16_t* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bins = 1 << bits;
    for (int i = threadIdx.x; i < WAVES * bins / 2; i += THREADS) reinterpret_cast<uint32_t*>(count)[i] = 0;
    __syncthreads();
    volatile uint16_t* mine = count + wave * bins;
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const uint32_t digit = digit_of(key[r], shift, bits);
        uint64_t same = ~0ull;
        for (int b = 0; b < bits; b++) {
            const bool set = digit >> b & 1;
            const uint64_t vote = __ballot(set);
            same &= set ? vote : ~vote;
        }
        const uint16_t before = mine[digit];
        rank[r] = before + __popcll(same & below);
        if ((same & below) == 0) mine[digit] = before + __popcll(same);  // (a wave's LDS operations keep their order)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += THREADS) {
        uint32_t sum = 0;
        for (int w = 0; w < WAVES; w++) {
            const uint16_t n = count[w * bins + d];
            count[w * bins + d] = sum;
            sum += n;
        }
        all[d] = sum;
    }
    __syncthreads();
}

// exclusive prefix sums of x over the workgroup (x of thread t in, sum of threads < t out)
__device__ __forceinline__ uint32_t before_me(uint32_t x, uint32_t* waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t sum = x;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(sum, o, 64);
        if (lane >= o) sum += y;
    }
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    uint32_t first = 0;
    for (int w = 0; w < wave; w++) first += waves[w];
    __syncthreads();
    return first + sum - x;
}

// zeros over `bytes` (from an address aligned to 2), by workgroups b of n
__device__ __forceinline__ void fill(void* p, long bytes, long b, long n) {
    uint8_t* at = static_cast<uint8_t*>(p);
    const long head = min((long)(-(uintptr_t)at & 15), bytes), quads = (bytes - head) / 16, tail = head + quads * 16;
    if (b == 0) {
        for (long i = threadIdx.x * 2; i < head; i += blockDim.x * 2) *reinterpret_cast<uint16_t*>(at + i) = 0;
        for (long i = tail + threadIdx.x * 2; i < bytes; i += blockDim.x * 2) *reinterpret_cast<uint16_t*>(at + i) = 0;
    }
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4* q = reinterpret_cast<u32x4*>(at + head);
    for (long i = b * blockDim.x + threadIdx.x; i < quads; i += n * blockDim.x) q[i] = u32x4{0, 0, 0, 0};
}

struct Fill {
    void* p;
    long bytes;
};

template <int ROUNDS>
__global__ __launch_bounds__(THREADS) void sort_fill(int M, long V, long skip, Digits dg, const int64_t* __restrict__ ids,
                                                     uint32_t* __restrict__ keys, uint32_t* __restrict__ places, Fill f) {
    __shared__ uint32_t key_lds[ROUNDS * THREADS];
    __shared__ uint16_t place_lds[ROUNDS * THREADS];
    __shared__ __attribute__((aligned(16))) uint16_t count[WAVES << MAX_BITS];
    __shared__ uint16_t all[1 << MAX_BITS];
    __shared__ uint32_t waves[WAVES];
    if (blockIdx.x > 0) {
        fill(f.p, f.bytes, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = wave * 64 * ROUNDS + lane;
    uint32_t key[ROUNDS];
    uint32_t place[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const int i = first + 64 * r;
        key[r] = i < M ? key_of(ids[i], V, skip) : ~0u;  // (behind all others: no key is larger in any digit)
        place[r] = i;
    }
    for (int p = 0; p < dg.passes; p++) {
        rank_digits<ROUNDS>(key, rank, p * dg.bits, dg.bits, count, all);
        const uint32_t n = threadIdx.x < 1u << dg.bits ? all[threadIdx.x] : 0, base = before_me(n, waves);
        if (threadIdx.x < 1u << dg.bits) all[threadIdx.x] = base;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint32_t digit = digit_of(key[r], p * dg.bits, dg.bits), to = (uint32_t)all[digit] + count[(wave << dg.bits) + digit] + rank[r];
            key_lds[to] = key[r];
            place_lds[to] = place[r];
            __builtin_amdgcn_sched_barrier(0);  // (not all rounds' addresses at once: registers)
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) key[r] = key_lds[first + 64 * r], place[r] = place_lds[first + 64 * r];
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const int i = first + 64 * r;
        if (i < M) keys[i] = key[r], places[i] = place[r];
    }
}

// One digit of a sort by many workgroups, BLOCK values each.  The first digit's values are the
// tokens themselves (from == nullptr).
struct Pass {
    long M, V, skip;
    int bits, shift, blocks;
    const int64_t* ids;
    const uint32_t *keys, *places;  // in (nullptr: the tokens)
    uint32_t *keys_out, *places_out;
    uint32_t* counts;  // [bins][blocks]
    uint32_t* totals;  // [bins]
};
__device__ __forceinline__ uint32_t key_at(const Pass& p, long i) { return p.keys ? p.keys[i] : key_of(p.ids[i], p.V, p.skip); }

__global__ __launch_bounds__(THREADS) void count_digits(Pass p, Fill f) {
    __shared__ uint32_t bins[1 << MAX_BITS];
    if ((int)blockIdx.x >= p.blocks) {
        fill(f.p, f.bytes, (int)blockIdx.x - p.blocks, (int)gridDim.x - p.blocks);
        return;
    }
    for (int d = threadIdx.x; d < 1 << p.bits; d += THREADS) bins[d] = 0;
    __syncthreads();
    const long first = (long)blockIdx.x * BLOCK;
#pragma unroll
    for (int r = 0; r < BLOCK / THREADS; r++) {
        const long i = first + r * THREADS + threadIdx.x;
        if (i < p.M) atomicAdd(&bins[digit_of(key_at(p, i), p.shift, p.bits)], 1u);  // (counts: their order changes nothing)
    }
    __syncthreads();
    for (int d = threadIdx.x; d < 1 << p.bits; d += THREADS) p.counts[(long)d * p.blocks + blockIdx.x] = bins[d];
}

// each digit's counts -> how many of it lie in the blocks before, and in all
__global__ __launch_bounds__(THREADS) void sum_counts(Pass p) {
    __shared__ uint32_t waves[WAVES];
    __shared__ uint32_t last;
    uint32_t* c = p.counts + (long)blockIdx.x * p.blocks;
    uint32_t sum = 0;
    for (int b0 = 0; b0 < p.blocks; b0 += THREADS) {
        const int b = b0 + threadIdx.x;
        const uint32_t n = b < p.blocks ? c[b] : 0, mine = sum + before_me(n, waves);
        if (b < p.blocks) c[b] = mine;
        if (threadIdx.x == THREADS - 1) last = mine + n;
        __syncthreads();
        sum = last;
        __syncthreads();
    }
    if (threadIdx.x == 0) p.totals[blockIdx.x] = sum;
}

__global__ __launch_bounds__(THREADS) void place_digits(Pass p) {
    constexpr int ROUNDS = BLOCK / THREADS;
    __shared__ __attribute__((aligned(16))) uint16_t count[WAVES << MAX_BITS];
    __shared__ uint16_t all[1 << MAX_BITS];
    __shared__ uint32_t base[1 << MAX_BITS];
    __shared__ uint32_t waves[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long first = (long)blockIdx.x * BLOCK + wave * 64 * ROUNDS + lane;
    uint32_t key[ROUNDS], place[ROUNDS];
    uint32_t rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const long i = first + 64 * r;
        key[r] = i < p.M ? key_at(p, i) : ~0u;  // (the last of their digit, and not placed)
        place[r] = i < p.M && p.places ? p.places[i] : (uint32_t)i;
    }
    const bool bin = threadIdx.x < 1u << p.bits;
    const uint32_t digit_first = before_me(bin ? p.totals[threadIdx.x] : 0, waves);
    if (bin) base[threadIdx.x] = digit_first + p.counts[(long)threadIdx.x * p.blocks + blockIdx.x];
    rank_digits<ROUNDS>(key, rank, p.shift, p.bits, count, all);
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        if (first + 64 * r >= p.M) continue;
        const uint32_t digit = digit_of(key[r], p.shift, p.bits), to = base[digit] + count[(wave << p.bits) + digit] + rank[r];
        p.keys_out[to] = key[r];
        p.places_out[to] = place[r];
    }
}

// ------------------------------------------------------------------------------ sums
struct Runs {
    long M, V;
    int D, each, slabs;  // each: tokens of a run; slabs: of a workgroup's columns
    long ldg;
    float scale;
};
struct Run {
    long from, to;
    bool inside, open;  // begins inside a stretch; ends inside one
};
__device__ __forceinline__ Run run_at(const Runs& s, const uint32_t* __restrict__ keys, long c) {
    Run r;
    r.from = c * s.each, r.to = min(r.from + s.each, s.M);
    r.inside = r.from > 0 && keys[r.from - 1] == keys[r.from];
    r.open = r.to < s.M && keys[r.to - 1] == keys[r.to];
    return r;
}

// (keys and places through pointers of their own: scalar loads, the same for a whole workgroup)
// parts: [run][2][D], of the stretch that a run begins inside of, of the one that it begins and does not end
template <int N, int BATCH, typename G, typename W>
__global__ __launch_bounds__(256) void sum_runs(Runs s, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ places,
                                                const G* __restrict__ grad, float* __restrict__ parts, W* __restrict__ dweight) {
    const int c = blockIdx.x / s.slabs, chunk = (blockIdx.x - c * s.slabs) * blockDim.x + threadIdx.x;
    if (chunk * N >= s.D) return;
    const int col = column<N>(chunk, s.D);
    const Run r = run_at(s, keys, c);
    if (keys[r.from] >= s.V) return;  // (sorted: nothing in this run counts)
    bool inside = r.inside;
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; e++) sum[e] = 0.f;
    for (long i0 = r.from; i0 < r.to; i0 += BATCH) {
        uint32_t key[BATCH + 1];
        float x[BATCH][N];
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
            const long i = min(i0 + j, r.to - 1);
            key[j] = keys[i];
            // (a token that adds nothing is not loaded: the run's first one is instead; streamed, 168 MB of
            // them and the rest 239 -> 224 us)
            load<N, true>(x[j], grad + (long)(key[j] < s.V ? places[i] : places[r.from]) * s.ldg + col);
        }
        key[BATCH] = keys[min(i0 + BATCH, s.M - 1)];
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
            if (i0 + j >= r.to || key[j] >= s.V) return;
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] += x[j][e];
            const bool end = i0 + j + 1 == r.to;
            if (!end && key[j + 1] == key[j]) continue;
            if (inside || (end && r.open)) {
                store<N>(parts + (2l * c + !inside) * s.D + col, sum);
            } else {
#pragma unroll
                for (int e = 0; e < N; e++) sum[e] *= s.scale;
                store<N>(dweight + (long)key[j] * s.D + col, sum);
            }
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] = 0.f;
            inside = false;
        }
    }
}

template <int N, typename W>
__global__ __launch_bounds__(256) void add_parts(Runs s, const uint32_t* __restrict__ keys, const float* __restrict__ parts,
                                                 W* __restrict__ dweight) {
    const int c = blockIdx.x / s.slabs, chunk = (blockIdx.x - c * s.slabs) * blockDim.x + threadIdx.x;
    const Run r = run_at(s, keys, c);
    const uint32_t key = keys[r.to - 1];
    if (!r.open || key >= s.V || (r.inside && keys[r.from] == key)) return;  // no stretch begins here and goes on
    // the last run that begins inside the stretch: 64 of them looked at together
    const int runs = (int)((s.M + s.each - 1) / s.each);
    int last = c;
    for (uint64_t same = ~0ull; same == ~0ull;) {
        const int d = last + 1 + (threadIdx.x & 63);
        same = __ballot(d < runs && keys[(long)d * s.each] == key);
        last += same == ~0ull ? 64 : __builtin_ctzll(~same);  // (sorted: those of the stretch come first)
    }
    if (chunk * N >= s.D) return;
    const int col = column<N>(chunk, s.D);
    float sum[N];
    load<N>(sum, parts + (2l * c + 1) * s.D + col);
    constexpr int BATCH = 8;
    for (int d0 = c + 1; d0 <= last; d0 += BATCH) {
        float x[BATCH][N];
#pragma unroll
        for (int j = 0; j < BATCH; j++) load<N>(x[j], parts + 2l * min(d0 + j, last) * s.D + col);
#pragma unroll
        for (int j = 0; j < BATCH; j++)
            if (d0 + j <= last)
#pragma unroll
                for (int e = 0; e < N; e++) sum[e] += x[j][e];
    }
#pragma unroll
    for (int e = 0; e < N; e++) sum[e] *= s.scale;
    store<N>(dweight + (long)key * s.D + col, sum);
}

// ------------------------------------------------------------------------------ few tokens
// One launch, no workspace: a workgroup has `rows` of the table's rows, writes their zeros, looks through all tokens for
// theirs, sorts those few by counting, and writes the rows that have some again.  `lanes` threads cover a row's columns (256 N
// of them at a time), and the 256 / lanes groups of threads take the rows in turn; a row of more than ALONE
// tokens is shared by the groups, their sums added in order: at most ALONE batches of BATCH tokens each.
// Bound by the zeros (200 tokens, 32768 x 2560 float32 with its lookup: 68 us, the zeros alone 49; rows written one by one,
// zeros or sums, in slabs of 256 chunks: 101) or, of small tables, by latency (512 tokens, 8192 x 256: 7.4 us).
constexpr int MOST = 1024;  // tokens
constexpr int ROWS = 256;   // of a workgroup
constexpr int ALONE = 16, BATCH = 16;

struct FewTokens {
    int M;
    long V, skip;
    int D, rows, lanes;
    long ldg;
    float scale;
};
template <int N, typename G, typename W>
__global__ __launch_bounds__(256) void few_tokens(FewTokens s, const int64_t* __restrict__ ids, const G* __restrict__ grad, W* __restrict__ dweight) {
    __shared__ uint16_t place[MOST], row[MOST], sorted[MOST];
    __shared__ int count[ROWS], start[ROWS];
    __shared__ int found[MOST / 64];
    __shared__ uint16_t present[ROWS];  // the rows that have tokens
    __shared__ int waves[4];
    __shared__ float parts[256 * N];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const long v0 = (long)blockIdx.x * s.rows;
    const int rows = (int)min((long)s.rows, s.V - v0);
    fill(dweight + v0 * s.D, (long)rows * s.D * sizeof(W), 0, 1);
    // this workgroup's tokens, in their order
    int mine[MOST / 256];
    uint64_t votes[MOST / 256];
#pragma unroll
    for (int j = 0; j < MOST / 256; j++) {
        const int i = 256 * j + t;
        const int64_t id = i < s.M ? ids[i] : -1;
        mine[j] = id >= v0 && id < v0 + rows && id != s.skip ? (int)(id - v0) : -1;
    }
#pragma unroll
    for (int j = 0; j < MOST / 256; j++) {
        votes[j] = __ballot(mine[j] >= 0);
        if (lane == 0) found[4 * j + wave] = __popcll(votes[j]);
    }
    count[t] = 0;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int k = 0; k < MOST / 64; k++) {
        if ((k & 3) == wave && mine[k >> 2] >= 0) {
            const int to = n + __popcll(votes[k >> 2] & ((1ull << lane) - 1));
            place[to] = 256 * (k >> 2) + t, row[to] = mine[k >> 2];
            atomicAdd(&count[mine[k >> 2]], 1);  // (counts: their order changes nothing)
        }
        n += found[k];
    }
    __syncthreads();
    if (n == 0) return;
    const uint64_t some = __ballot(count[t] > 0);
    if (lane == 0) waves[wave] = __popcll(some);
    if (count[t] > 0) {
        int before = 0;
        for (int k = 0; k < t; k++) before += count[k];
        start[t] = before;
    }
    __syncthreads();
    int all = 0, at_row = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) at_row += w < wave ? waves[w] : 0, all += waves[w];
    if (count[t] > 0) present[at_row + __popcll(some & ((1ull << lane) - 1))] = t;
    for (int i = t; i < n; i += 256) {
        int before = start[row[i]];
        for (int k = 0; k < i; k++) before += row[k] == row[i];
        sorted[before] = place[i];
    }
    __syncthreads();
    const int groups = 256 / s.lanes, group = t / s.lanes, at = t - group * s.lanes;
    for (int c0 = 0; c0 * N < s.D; c0 += 256) {
        const int chunk = c0 + at;
        const bool there = chunk * N < s.D;
        const int col = column<N>(there ? chunk : 0, s.D);
        auto sum_of = [&](float (&sum)[N], int from, int to) {
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] = 0.f;
            for (int i0 = from; i0 < to; i0 += BATCH) {
                float x[BATCH][N];
#pragma unroll
                for (int j = 0; j < BATCH; j++) load<N, true>(x[j], grad + (long)sorted[min(i0 + j, to - 1)] * s.ldg + col);
#pragma unroll
                for (int j = 0; j < BATCH; j++)
                    if (i0 + j < to)
#pragma unroll
                        for (int e = 0; e < N; e++) sum[e] += x[j][e];
            }
        };
        auto put = [&](int r, float (&sum)[N]) {
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] *= s.scale;
            store<N>(dweight + (v0 + r) * s.D + col, sum);
        };
        if (there)
            for (int k = group; k < all; k += groups) {
                const int r = present[k];
                if (count[r] > ALONE) continue;
                float sum[N];
                sum_of(sum, start[r], start[r] + count[r]);
                put(r, sum);
            }
        if (n <= ALONE) continue;
        for (int k = 0; k < all; k++) {
            const int r = present[k], c = count[r];
            if (c <= ALONE) continue;
            const int each = (c + groups - 1) / groups, from = start[r] + min(group * each, c), to = start[r] + min(group * each + each, c);
            float sum[N];
            sum_of(sum, from, to);
            __syncthreads();
#pragma unroll
            for (int e = 0; e < N; e++) parts[N * t + e] = sum[e];
            __syncthreads();
            if (group == 0 && there) {
                for (int g = 1; g < groups; g++)
#pragma unroll
                    for (int e = 0; e < N; e++) sum[e] += parts[N * (g * s.lanes + at) + e];
                put(r, sum);
            }
        }
    }
}

// ------------------------------------------------------------------------------ host
static int check(long M, long V, int D) {
    return M < 0 || M > (1l << 30) || V < 1 || V > (1l << 22) || D < 1 || D > (1 << 17) ? THESEUS_WKV7_ERR_SHAPE : THESEUS_WKV7_OK;
}
template <class Go> static void with_types(int from, int to, Go go) {
    if (from == THESEUS_EMBED_BF16) {
        if (to == THESEUS_EMBED_BF16) go(uint16_t{}, uint16_t{});
        else go(uint16_t{}, float{});
    } else {
        if (to == THESEUS_EMBED_BF16) go(float{}, uint16_t{});
        else go(float{}, float{});
    }
}
static bool known(int dtype) { return dtype == THESEUS_EMBED_BF16 || dtype == THESEUS_EMBED_FP32; }

struct Plan {
    long runs, blocks;
    int each;
    size_t keys, places, keys2, places2, counts, totals, parts, bytes;
};
static Plan plan(long M, long V, int D) {
    Plan p{};
    p.each = 16;  // (shorter ones leave more parts, longer ones too few workgroups; from 32768 tokens on 2048 runs)
    while (p.each * 2048l < M) p.each *= 2;
    p.runs = ceil_div(M, p.each);
    p.blocks = M > ONE ? ceil_div(M, BLOCK) : 0;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) / 256 * 256;
        return here;
    };
    p.keys = take(M * 4), p.places = take(M * 4);
    if (p.blocks) {
        p.keys2 = take(M * 4), p.places2 = take(M * 4);
        p.counts = take((size_t)p.blocks * 4 << digits(V).bits);
        p.totals = take((size_t)4 << digits(V).bits);
    }
    p.parts = take((size_t)p.runs * 2 * D * 4);
    p.bytes = at;
    return p;
}

// threads for a row's columns; whether few_tokens takes this many tokens: as many as its LDS and its batches for one row hold.
// Against the sort and sums (float32 tables, us): 8192 x 256 with 16 tokens 6.1 and 14.3, 512 8.4 and 17.9, 1024 10.1 and 18.3;
// 65536 x 256 with 1024 17.5 and 21.7; 8192 x 2560 with 256 23.1 and 24.2, 8192 x 5120 with 256 37.2 and 34.7; tables whose zeros
// take longer the same either way.
static int lanes_of(int D) {
    const long chunks = D >= 8 ? ceil_div(D, 8) : D;
    int lanes = 1;
    while (lanes < 256 && lanes < chunks) lanes *= 2;
    return lanes;
}
static bool is_few(long M, int D) { return M <= MOST && M <= ALONE * BATCH * (256 / lanes_of(D)); }

template <int N, typename G, typename W>
static void launch_few(FewTokens s, const int64_t* ids, const void* grad, void* dweight, hipStream_t st) {
    s.lanes = lanes_of(s.D);
    // rows for about four workgroups on a CU, of at most 64 KB
    const long share = ceil_div(s.V, 1024), most = 65536 / (s.D * (long)sizeof(W)), least = share < most ? share : most;
    s.rows = (int)(least < 1 ? 1 : least > ROWS ? ROWS : least);
    few_tokens<N, G, W><<<(unsigned)ceil_div(s.V, s.rows), 256, 0, st>>>(s, ids, static_cast<const G*>(grad), static_cast<W*>(dweight));
}

template <int N, typename W, typename O>
static void launch_lookup(long M, long V, int D, const int64_t* ids, const void* w, long ldw, float scale, void* out, hipStream_t st) {
    const long chunks = M * ceil_div(D, N);
    auto go = [&](auto each) {
        constexpr int EACH = decltype(each)::value;
        const long blocks = ceil_div(chunks, 256 * EACH);
        lookup<N, EACH><<<(unsigned)(blocks < 1 << 20 ? blocks : 1 << 20), 256, 0, st>>>(M, V, D, ids, static_cast<const W*>(w), ldw, scale,
                                                                                    static_cast<O*>(out));
    };
    if (chunks < 256 * 2048) go(std::integral_constant<int, 1>{});  // (a workgroup for every wave slot first, then loads in flight)
    else go(std::integral_constant<int, 4>{});
}

template <int N, typename G, typename W>
static void launch_sums(Runs s, long runs, const uint32_t* keys, const uint32_t* places, const void* grad, float* parts, void* dweight,
                        hipStream_t st) {
    const long chunks = ceil_div(s.D, N);
    const int threads = chunks >= 256 ? 256 : (int)(ceil_div(chunks, 64) * 64);
    s.slabs = (int)ceil_div(chunks, threads);
    const unsigned grid = (unsigned)(runs * s.slabs);
    sum_runs<N, 32 / sizeof(G), G, W><<<grid, threads, 0, st>>>(s, keys, places, static_cast<const G*>(grad), parts, static_cast<W*>(dweight));
    if (runs > 1) add_parts<N, W><<<grid, threads, 0, st>>>(s, keys, parts, static_cast<W*>(dweight));
}

}  // namespace embed

extern "C" {

int theseus_embed_lookup(long long M, long long V, int D, int weight_dtype, int out_dtype, const int64_t* ids, const void* weight,
                         long long weight_stride, float scale, void* out, hipStream_t stream) {
    if (int e = embed::check(M, V, D)) return e;
    if (V > 1 && weight_stride < D) return THESEUS_WKV7_ERR_SHAPE;
    if (!embed::known(weight_dtype) || !embed::known(out_dtype)) return THESEUS_WKV7_ERR_DTYPE;
    if (M == 0) return THESEUS_WKV7_OK;
    if (!ids || !weight || !out) return THESEUS_WKV7_ERR_NULL;
    auto go = [&](auto w, auto o) {
        using W = decltype(w);
        using O = decltype(o);
        if (D >= 8) embed::launch_lookup<8, W, O>(M, V, D, ids, weight, weight_stride, scale, out, stream);
        else embed::launch_lookup<1, W, O>(M, V, D, ids, weight, weight_stride, scale, out, stream);
    };
    embed::with_types(weight_dtype, out_dtype, go);
    return hipGetLastError() == hipSuccess ? THESEUS_WKV7_OK : THESEUS_WKV7_ERR_LAUNCH;
}

size_t theseus_embed_grad_workspace_size(long long M, long long V, int D) {
    return embed::check(M, V, D) || embed::is_few(M, D) ? 0 : embed::plan(M, V, D).bytes;
}

int theseus_embed_grad(long long M, long long V, int D, int grad_dtype, int weight_dtype, const int64_t* ids, long long skip,
                       const void* grad, long long grad_stride, float scale, void* dweight, void* workspace, size_t workspace_bytes,
                       hipStream_t stream) {
    using namespace embed;
    if (int e = check(M, V, D)) return e;
    if (M > 1 && grad_stride != 0 && grad_stride < D) return THESEUS_WKV7_ERR_SHAPE;
    if (!known(grad_dtype) || !known(weight_dtype)) return THESEUS_WKV7_ERR_DTYPE;
    if (!dweight || (M && (!ids || !grad))) return THESEUS_WKV7_ERR_NULL;
    if (is_few(M, D)) {
        const FewTokens s{(int)M, V, skip, D, 0, 0, grad_stride, scale};
        with_types(grad_dtype, weight_dtype, [&](auto g, auto w) {
            using G = decltype(g);
            using W = decltype(w);
            if (D >= 8) launch_few<8, G, W>(s, ids, grad, dweight, stream);
            else launch_few<1, G, W>(s, ids, grad, dweight, stream);
        });
        return hipGetLastError() == hipSuccess ? THESEUS_WKV7_OK : THESEUS_WKV7_ERR_LAUNCH;
    }
    const Plan p = plan(M, V, D);
    if (!workspace || workspace_bytes < p.bytes) return THESEUS_WKV7_ERR_WORKSPACE;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    auto at = [&](size_t off) { return reinterpret_cast<uint32_t*>(ws + off); };
    const Digits dg = digits(V);
    const Fill f{dweight, V * D * (weight_dtype == THESEUS_EMBED_BF16 ? 2l : 4l)};
    // four stores a thread: enough workgroups that some are always starting (671 MB behind a sort of 16384 tokens, the whole
    // gradient with its lookup: 281 us with 1024 of them, 242 with 8192, 239 so)
    const long want = ceil_div(f.bytes, THREADS * 16 * 4), fills = want < 1 << 21 ? want : 1 << 21;
    const uint32_t *keys = at(p.keys), *places = at(p.places);
    if (M <= ONE) {
        auto sort = [&](auto rounds) {
            sort_fill<decltype(rounds)::value><<<(unsigned)(1 + fills), THREADS, 0, stream>>>((int)M, V, skip, dg, ids, at(p.keys), at(p.places), f);
        };
        // (rounds for all of ONE whatever M: 2048 tokens, 8192 x 256, 39 us for 19, 4096 40 for 22, 6144 41 for 26)
        if (M <= 2 * THREADS) sort(std::integral_constant<int, 2>{});
        else if (M <= 4 * THREADS) sort(std::integral_constant<int, 4>{});
        else if (M <= 6 * THREADS) sort(std::integral_constant<int, 6>{});
        else sort(std::integral_constant<int, ONE / THREADS>{});
    } else {
        Pass q{M, V, skip, dg.bits, 0, (int)p.blocks, ids, nullptr, nullptr, at(p.keys), at(p.places), at(p.counts), at(p.totals)};
        for (int i = 0; i < dg.passes; i++) {
            q.shift = i * dg.bits;
            count_digits<<<(unsigned)(p.blocks + (i == 0 ? fills : 0)), THREADS, 0, stream>>>(q, f);
            sum_counts<<<1u << dg.bits, THREADS, 0, stream>>>(q);
            place_digits<<<(unsigned)p.blocks, THREADS, 0, stream>>>(q);
            keys = q.keys_out, places = q.places_out;
            q.keys = keys, q.places = places;
            const bool second = keys == at(p.keys);
            q.keys_out = at(second ? p.keys2 : p.keys), q.places_out = at(second ? p.places2 : p.places);
        }
    }
    {
        const Runs s{M, V, D, p.each, 0, grad_stride, scale};
        float* parts = reinterpret_cast<float*>(ws + p.parts);
        auto go = [&](auto g, auto w) {
            using G = decltype(g);
            using W = decltype(w);
            if (D >= 8) launch_sums<8, G, W>(s, p.runs, keys, places, grad, parts, dweight, stream);
            else launch_sums<1, G, W>(s, p.runs, keys, places, grad, parts, dweight, stream);
        };
        with_types(grad_dtype, weight_dtype, go);
    }
    return hipGetLastError() == hipSuccess ? THESEUS_WKV7_OK : THESEUS_WKV7_ERR_LAUNCH;
}

}  // extern "C"
