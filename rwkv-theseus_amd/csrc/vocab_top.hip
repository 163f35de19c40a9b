// The k largest logits of each row with their indices, and the row's log-sum-exp, in one pass
// over the logits (C ABI: include/theseus_vocab.h).
//
// A workgroup of 1024 threads takes up to SLAB elements of a row into registers (128 KB read once)
// and selects there:
//   1. every thread's maximum and, against the row's, its sum of exponentials;
//   2. the k-th largest of 256 (k <= 128) or 512 group maxima, rounded down to 16 bits, is a bound that the k-th largest
//      element cannot be below: -G ln(1 - k/G) elements (74 of 65536 for k = 64, 355 for k = 256)
//      are not below it in independent data;
//   3. the elements not below the bound go to a list in LDS as (key, ~index) in 64 bits, whose
//      order is the answer's; each one's rank is a count over the list (of more than MANY, over
//      those that are not below its k-th key, found by bisection).
// With more than CAP elements at the bound (many equal values: a masked vocabulary), the list
// takes those above it, and of the equal ones those of the lowest indices, found by bisection on
// the index; should more than CAP lie above it, the exact k-th key is found by bisection first.
// Rows longer than a slab are cut into slabs whose sorted lists top_merge joins, MERGE at a time.
//
// Keys order like the values: NaN above all, -0 as +0; 0 stands for "no element".
#include "../../include/theseus_vocab.h"
#include "../../include/theseus_wkv7.h"

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "wkv7_common.h"

namespace vocab_top {

constexpr int THREADS = 1024, SMALL = 256;  // of a workgroup
constexpr int MOST = 8;                     // 16-byte granules per thread
constexpr int MANY = 256;                   // list entries worth another selection
constexpr int MERGE = 16;    // lists joined at a time
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t u = __float_as_uint(f + 0.f);
    return f != f ? 0xffffffffu : (int32_t)u < 0 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((int32_t)k < 0 ? k & 0x7fffffffu : ~k); }

// what a row's exponentials are taken against (an infinite maximum would leave inf - inf)
__device__ __forceinline__ float base_of(float top) { return fabsf(top) == INFINITY ? 0.f : top; }

struct Args {
    long rows, vocab, stride;
    int k, slabs, each;     // slabs of a row, granules of a slab
    float scale, inv_T;     // log2(e) / temperature, 1 / temperature
    const void* x;
    void* values;           // slabs == 1: the answer
    int64_t* indices;
    float* lse;
    uint64_t* lists;        // slabs > 1: [rows][slabs][k]
    float2* sums;           // [rows][slabs] {maximum, sum of exponentials against it}
};

// (the value comes out of the key, without reading the logit again: -0 as 0, any NaN as one)
template <bool BF16> __device__ __forceinline__ void emit(const Args& p, long row, int rank, uint64_t c) {
    const long at = row * p.k + rank;
    const uint32_t u = __float_as_uint(of_key((uint32_t)(c >> 32)));
    p.indices[at] = 0xffffffffu - (uint32_t)c;
    if constexpr (BF16) static_cast<uint16_t*>(p.values)[at] = (uint16_t)(u >> 16);
    else static_cast<uint32_t*>(p.values)[at] = u;
}

// A workgroup of T threads, G granules each: slabs of at most T G granules.  (8 waves a SIMD, 64
// registers: two workgroups of 1024 on a CU, one loading while the other selects; 4096 rows of
// 65536 bfloat16 180 -> 126 us.)  T = 1024, or 256 with k <= 128.
template <bool BF16, int T, int G> __global__ __launch_bounds__(T, 8) void top_part(Args p) {
    constexpr int PER = BF16 ? 8 : 4;  // elements of a granule
    constexpr int WAVES = T / 64, CAP = T, GROUPS = T < 512 ? T : 512, KEYS = CAP / 64;
    __shared__ __attribute__((aligned(16))) uint64_t list[CAP];
    __shared__ __attribute__((aligned(16))) float maxima[GROUPS];
    __shared__ int ranks[CAP];
    __shared__ float shared_bound;
    __shared__ uint32_t shared_key;
    __shared__ float redf[2][WAVES];
    __shared__ int count;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const long row = blockIdx.x / p.slabs;
    const int slab = blockIdx.x - row * p.slabs;

    // Granules are 16-byte aligned in memory, whatever the row's alignment: a row's first and last
    // may hold elements of a neighbour (or of the allocation that the row lies in, which starts
    // and ends on such a granule), left out below.  Slab s has granules s each .. of the row.
    const long size = BF16 ? 2 : 4;
    const uint8_t* row0 = static_cast<const uint8_t*>(p.x) + row * p.stride * size;
    const int shift = (int)((uintptr_t)row0 & 15) / (int)size, V = (int)p.vocab;  // elements of the first granule before the row
    const int gall = (V + shift + PER - 1) / PER, g0 = slab * p.each, gend = min(g0 + p.each, gall);
    const uint4* gran = reinterpret_cast<const uint4*>(row0 - shift * size);
    uint32_t w[G][4];
#pragma unroll
    for (int j = 0; j < G; j++) {
        const uint4 u = gran[min(g0 + j * T + t, gend - 1)];
        w[j][0] = u.x, w[j][1] = u.y, w[j][2] = u.z, w[j][3] = u.w;
    }
    if (t == 0) count = 0;
    auto val = [](const uint32_t (&u)[4], int e) {  // element e of a granule
        if constexpr (BF16) return __uint_as_float(e & 1 ? u[e >> 1] & 0xffff0000u : u[e >> 1] << 16);
        else return __uint_as_float(u[e]);
    };
    constexpr uint32_t LOW = BF16 ? 0xff80ff80u : 0xff800000u;
    if ((g0 == 0 && shift) || gend == gall || p.each < T * G) {  // (elsewhere every element is the slab's)
#pragma unroll
        for (int j = 0; j < G; j++) {
            const int g = g0 + j * T + t;
            const bool out = g >= gend;
#pragma unroll
            for (int i = 0; i < 4; i++) w[j][i] = out ? LOW : w[j][i];
            if ((g == 0 && shift) || (g == gall - 1 && (V + shift) % PER)) {
#pragma unroll
                for (int e = 0; e < PER; e++) {
                    const int i = g * PER + e - shift;
                    if (i < 0 || i >= V) {
                        if constexpr (BF16) w[j][e >> 1] = e & 1 ? (w[j][e >> 1] & 0xffffu) | 0xff800000u : (w[j][e >> 1] & 0xffff0000u) | 0xff80u;
                        else w[j][e] = 0xff800000u;
                    }
                }
            }
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < G; j++)
#pragma unroll
        for (int e = 0; e < PER; e++) top = fmaxf(top, val(w[j], e));
    // groups of four threads, of two for k > 128; the small workgroup's threads
    const int lg = T == SMALL ? 0 : p.k > 128 ? 1 : 2;
    float all = top;
    if (lg > 0) all = fmaxf(all, __shfl_xor(all, 1, 64));
    if (lg == 2) all = fmaxf(all, __shfl_xor(all, 2, 64));
    if ((t & ((1 << lg) - 1)) == 0) maxima[t >> lg] = all;
    ranks[t] = 0;
    for (int o = 32; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o, 64));
    if (lane == 0) redf[0][wave] = all;
    __syncthreads();
    for (int i = 0; i < WAVES; i++) all = fmaxf(all, redf[0][i]);

    const float base = base_of(all), b = base * p.scale;
    float sum = 0.f;
    // x scale - b is one fma, whose exponents are all off by b's rounding, as the lse is by that of its own
    // largest part: up to 2^12 that shift is below 2^-12.  Beyond, where it would reach whole powers of two (and the
    // products overflow at the type's ends), the difference is taken first: the maximum's term is 1.  (One operation
    // more for each element.)
    if (fabsf(b) < 4096.f) {
#pragma unroll
        for (int j = 0; j < G; j++)
#pragma unroll
            for (int e = 0; e < PER; e++) sum += __builtin_amdgcn_exp2f(val(w[j], e) * p.scale - b);
    } else {
#pragma unroll
        for (int j = 0; j < G; j++)
#pragma unroll
            for (int e = 0; e < PER; e++) sum += __builtin_amdgcn_exp2f((val(w[j], e) - base) * p.scale);
    }
    const bool nan = sum != sum;  // (a thread with a NaN among its elements, or nearly so: it looks at all of them)
    float s = sum;
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) redf[1][wave] = s;

    if (wave == 0) {  // the k-th largest group maximum: the upper 16 bits of its key, by bisection
        uint32_t key[8];
#pragma unroll
        for (int i = 0; i < 4; i++) key[i] = key_of(maxima[64 * i + lane]);
#pragma unroll
        for (int i = 4; i < 8; i++) key[i] = GROUPS == 512 && lg == 1 ? key_of(maxima[(64 * i + lane) & (GROUPS - 1)]) : 0;
        uint32_t found = 0;
#pragma unroll 1
        for (int bit = 31; bit >= 16; bit--) {
            const uint32_t c = found | (1u << bit);
            int n = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) n += __popcll(__ballot(key[i] >= c));
            if (lg == 1)
#pragma unroll
                for (int i = 4; i < 8; i++) n += __popcll(__ballot(key[i] >= c));
            if (n >= p.k) found = c;
        }
        if (lane == 0) shared_bound = of_key(max(found, key_of(-INFINITY)));  // (fewer groups than k: everything)
    }
    __syncthreads();
    if (t == 0) {
        float total = 0.f;
        for (int i = 0; i < WAVES; i++) total += redf[1][i];
        if (p.slabs > 1) p.sums[row * p.slabs + slab] = make_float2(base, total);
        else if (p.lse) p.lse[row] = base * p.inv_T + __builtin_amdgcn_logf(total) * LN2;  // (nothing but -inf: log2 0)
    }
    const float bound = shared_bound;
    const uint32_t bk = key_of(bound);

    auto append = [&](int i, uint32_t key) {
        const int at = atomicAdd(&count, 1);
        if (at < CAP) list[at] = (uint64_t)key << 32 | (0xffffffffu - (uint32_t)i);
    };
    if (nan || !(top < bound)) {
        // the granules to look at, then each of them
        uint32_t hit = 0;
#pragma unroll
        for (int j = 0; j < G; j++) {
            float m = val(w[j], 0);
#pragma unroll
            for (int e = 1; e < PER; e++) m = fmaxf(m, val(w[j], e));
            hit |= (uint32_t)(nan || !(m < bound)) << j;
        }
        for (; hit; hit &= hit - 1) {
            const int j = __ffs(hit) - 1, g = g0 + j * T + t;
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = w[0][i];
#pragma unroll
            for (int jj = 1; jj < G; jj++)
#pragma unroll
                for (int i = 0; i < 4; i++) u[i] = jj == j ? w[jj][i] : u[i];
#pragma unroll
            for (int e = 0; e < PER; e++) {
                const int i = g * PER + e - shift;
                const float f = val(u, e);
                if (!(f < bound) && i >= 0 && i < V && g < gend) append(i, key_of(f));
            }
        }
    }
    __syncthreads();
    int n = count;
    if (n > CAP) {
        // f(index, key) for every element of the slab, read again
        auto each = [&](auto f) {
#pragma unroll 1
            for (int g = g0 + t; g < gend; g += T) {
                const uint4 q = gran[g];
                const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int e = 0; e < PER; e++) {
                    const int i = g * PER + e - shift;
                    if (i >= 0 && i < V) f(i, key_of(val(u, e)));
                }
            }
        };
        // how many elements f holds for (with a barrier before and after)
        auto counted = [&](auto f) {
            __syncthreads();
            if (t == 0) count = 0;
            __syncthreads();
            int c = 0;
            each([&](int i, uint32_t key) { c += f(i, key); });
            for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
            if (lane == 0) atomicAdd(&count, c);
            __syncthreads();
            return count;
        };
        uint32_t K = bk;
        int above = counted([&](int, uint32_t key) { return key > K; });
        if (above >= p.k) {  // (the bound was not the k-th key: find it)
            K = 0;
#pragma unroll 1
            for (int bit = 31; bit >= 0; bit--) {
                const uint32_t c = K | (1u << bit);
                if (counted([&](int, uint32_t key) { return key >= c; }) >= p.k) K = c;
            }
            above = counted([&](int, uint32_t key) { return key > K; });
        }
        // the k - above elements equal to K of the lowest indices: those up to `last`
        int last = 0;
#pragma unroll 1
        for (int bit = 30; bit >= 0; bit--) {
            const int c = last | (1 << bit);
            if (counted([&](int i, uint32_t key) { return key == K && i < c; }) < p.k - above) last = c;
        }
        __syncthreads();
        if (t == 0) count = 0;
        __syncthreads();
        each([&](int i, uint32_t key) {
            if (key > K || (key == K && i <= last)) append(i, key);
        });
        __syncthreads();
        n = count;
    }
    if (n > MANY) {  // (few values of one group are left out where they are fewer than the groups)
        const uint64_t c = t < n ? list[t] : 0;
        if (wave == 0) {  // the list's k-th key
            uint32_t key[KEYS], found = 0;
#pragma unroll
            for (int i = 0; i < KEYS; i++) key[i] = 64 * i + lane < n ? (uint32_t)(list[64 * i + lane] >> 32) : 0;
#pragma unroll 1
            for (int bit = 31; bit >= 0; bit--) {
                const uint32_t x = found | (1u << bit);
                int m = 0;
#pragma unroll
                for (int i = 0; i < KEYS; i++) m += __popcll(__ballot(key[i] >= x));
                if (m >= p.k) found = x;
            }
            if (lane == 0) shared_key = found;
        }
        __syncthreads();
        if (t == 0) count = 0;
        __syncthreads();
        if (t < n && (uint32_t)(c >> 32) >= shared_key) list[atomicAdd(&count, 1)] = c;
        __syncthreads();
        n = count;
    }
    int lanes = 64, ln = 6;  // threads of one share of the counting: a power of two, n at least
    while (lanes < n) lanes *= 2, ln++;
    const int own = t & (lanes - 1);
    const uint64_t c = own < n ? list[own] : 0;
    {
        const int shares = T >> ln, share = ((n + shares - 1) / shares + 1) & ~1, first = (t >> ln) * share;
        int r = 0;
        for (int i = first; i < min(n, first + share); i += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(list + i);
            r += (two.x > c) + (i + 1 < n && two.y > c);
        }
        if (own < n) atomicAdd(ranks + own, r);
    }
    __syncthreads();
    if (t < n && ranks[t] < p.k) {
        if (p.slabs > 1) p.lists[((long)row * p.slabs + slab) * p.k + ranks[t]] = c;
        else emit<BF16>(p, row, ranks[t], c);
    }
    if (p.slabs > 1)  // (a short last slab)
        for (int i = n + t; i < p.k; i += T) p.lists[((long)row * p.slabs + slab) * p.k + i] = 0;
}

// Joins up to MERGE sorted lists of a row: an entry's rank is its place in its own list and the
// numbers of greater entries in the others (bisection).  `last`: the answer, else a list again.
template <bool BF16> __global__ __launch_bounds__(THREADS) void top_merge(Args p, const uint64_t* in, int lists, uint64_t* out, int groups, int last) {
    __shared__ uint64_t c[MERGE * THESEUS_VOCAB_MAX_TOP];
    const long row = blockIdx.x / groups;
    const int g = blockIdx.x - row * groups, first = g * MERGE, nl = min(MERGE, lists - first), total = nl * p.k;
    const uint64_t* from = in + (row * lists + first) * p.k;
    for (int i = threadIdx.x; i < total; i += THREADS) c[i] = from[i];
    __syncthreads();
    for (int i = threadIdx.x; i < total; i += THREADS) {
        const uint64_t x = c[i];
        const int own = i / p.k;
        int rank = i - own * p.k;
        for (int l = 0; l < nl && rank < p.k; l++) {
            if (l == own) continue;
            const uint64_t* y = c + l * p.k;
            int lo = 0, hi = p.k;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                // (absent entries, all 0, go by their list: the answer never has one)
                if (y[mid] > x || (y[mid] == x && l < own)) lo = mid + 1;
                else hi = mid;
            }
            rank += lo;
        }
        if (rank < p.k) {
            if (last) emit<BF16>(p, row, rank, x);
            else out[(row * groups + g) * p.k + rank] = x;
        }
    }
    if (last && p.lse && threadIdx.x < 64) {
        const float2* s = p.sums + row * p.slabs;
        float top = -INFINITY, sum = 0.f;
        for (int i = threadIdx.x; i < p.slabs; i += 64)
            if (!(s[i].y == 0.f)) top = fmaxf(top, s[i].x);
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float b = top == -INFINITY ? 0.f : top;
        for (int i = threadIdx.x; i < p.slabs; i += 64)
            if (!(s[i].y == 0.f)) sum += s[i].y == INFINITY ? INFINITY : s[i].y * __builtin_amdgcn_exp2f((s[i].x - b) * p.scale);
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (threadIdx.x == 0) p.lse[row] = b * p.inv_T + __builtin_amdgcn_logf(sum) * LN2;
    }
}

static size_t up(size_t n) { return (n + 255) / 256 * 256; }
struct Plan {
    int threads, granules;  // per thread
    long slabs, each;       // of a row; granules of one
};
// The smallest slab that holds a row, or slabs of one size: a second slab costs its merge (4 us and,
// for one row of 65536 bfloat16, 12.2 us in two against 10.0 in one).  With enough rows to fill
// the CUs eight times over, short rows go to workgroups of 256 (4096 rows of 8192).
static Plan plan(long rows, long vocab, int k, int dtype, bool aligned) {
    const long per = dtype == THESEUS_VOCAB_BF16 ? 8 : 4;
    // (a row that does not start on a granule may have one more)
    const long all = (vocab + (aligned ? 0 : per - 1) + per - 1) / per;
    const int threads = rows >= 1024 && k <= 128 && all <= SMALL * MOST ? SMALL : THREADS;
    int g = 1;
    while (g < MOST && all > (long)threads * g) g *= 2;
    const long slabs = (all + (long)threads * g - 1) / ((long)threads * g);
    return {threads, g, slabs, (all + slabs - 1) / slabs};
}
static size_t bytes_of(size_t rows, size_t s, int k) {
    if (s == 1) return 0;
    const size_t groups = (s + MERGE - 1) / MERGE;
    return up(rows * s * k * 8) + up(rows * s * 8) + (groups > 1 ? up(rows * groups * k * 8) : 0);
}

static int check(long long rows, long long vocab, int k, int dtype) {
    if (rows < 0 || rows > (1ll << 30) || vocab < 1 || vocab > (1ll << 30) || k < 1 || k > vocab || k > THESEUS_VOCAB_MAX_TOP)
        return THESEUS_WKV7_ERR_SHAPE;
    if (dtype != THESEUS_VOCAB_BF16 && dtype != THESEUS_VOCAB_FP32) return THESEUS_WKV7_ERR_DTYPE;
    if (rows * plan(rows, vocab, k, dtype, false).slabs >= (1ll << 31)) return THESEUS_WKV7_ERR_SHAPE;
    return THESEUS_WKV7_OK;
}

template <bool BF16> static void launch(Args p, const Plan& pl, uint8_t* ws, hipStream_t st) {
    const size_t lists = up((size_t)p.rows * p.slabs * p.k * 8);
    p.lists = reinterpret_cast<uint64_t*>(ws);
    p.sums = reinterpret_cast<float2*>(ws + lists);
    const unsigned n = (unsigned)(p.rows * p.slabs);
    auto part = [&](auto tag) {
        constexpr int G = decltype(tag)::value;
        if (pl.threads == SMALL) top_part<BF16, SMALL, G><<<n, SMALL, 0, st>>>(p);
        else top_part<BF16, THREADS, G><<<n, THREADS, 0, st>>>(p);
    };
    switch (pl.granules) {
        case 1: part(std::integral_constant<int, 1>{}); break;
        case 2: part(std::integral_constant<int, 2>{}); break;
        case 4: part(std::integral_constant<int, 4>{}); break;
        default: part(std::integral_constant<int, MOST>{});
    }
    if (p.slabs == 1) return;
    uint64_t* in = p.lists;
    uint64_t* out = reinterpret_cast<uint64_t*>(ws + lists + up((size_t)p.rows * p.slabs * 8));
    for (int n = p.slabs;;) {
        const int groups = (n + MERGE - 1) / MERGE;
        top_merge<BF16><<<(unsigned)(p.rows * groups), THREADS, 0, st>>>(p, in, n, out, groups, groups == 1);
        if (groups == 1) return;
        uint64_t* t = in;
        in = out, out = t;
        n = groups;
    }
}

}  // namespace vocab_top

extern "C" {

size_t theseus_vocab_top_workspace_size(long long rows, long long vocab, int k, int dtype) {
    using namespace vocab_top;
    if (check(rows, vocab, k, dtype)) return 0;
    const size_t a = bytes_of((size_t)rows, (size_t)plan(rows, vocab, k, dtype, true).slabs, k);
    const size_t b = bytes_of((size_t)rows, (size_t)plan(rows, vocab, k, dtype, false).slabs, k);
    return a > b ? a : b;
}

int theseus_vocab_top(long long rows, long long vocab, int k, int dtype, float temperature, const void* logits,
                      long long row_stride, void* values, int64_t* indices, float* lse, void* workspace,
                      size_t workspace_bytes, hipStream_t stream) {
    using namespace vocab_top;
    if (int e = check(rows, vocab, k, dtype)) return e;
    if (row_stride < vocab || !(temperature > 0.f) || !isfinite(temperature)) return THESEUS_WKV7_ERR_SHAPE;
    if (!rows) return THESEUS_WKV7_OK;
    if (!logits || !values || !indices) return THESEUS_WKV7_ERR_NULL;
    const int size = dtype == THESEUS_VOCAB_BF16 ? 2 : 4;
    if ((uintptr_t)logits % size) return THESEUS_WKV7_ERR_SHAPE;
    const Plan pl = plan(rows, vocab, k, dtype, ((uintptr_t)logits | (uintptr_t)(row_stride * size)) % 16 == 0);
    const size_t need = bytes_of((size_t)rows, (size_t)pl.slabs, k);
    if (need && (!workspace || workspace_bytes < need)) return THESEUS_WKV7_ERR_WORKSPACE;
    // A launch has fewer than 2^32 threads: more rows than that (4 million of one slab) in several, in one workspace.
    const long most = (long)(0xffffffffu / THREADS) / pl.slabs;
    for (long r0 = 0; r0 < rows; r0 += most) {
        Args p{rows - r0 < most ? rows - r0 : most, vocab, row_stride, k, (int)pl.slabs, (int)pl.each, LOG2E / temperature, 1.f / temperature,
               static_cast<const uint8_t*>(logits) + r0 * row_stride * size, static_cast<uint8_t*>(values) + r0 * k * size,
               indices + r0 * k, lse ? lse + r0 : nullptr, nullptr, nullptr};
        if (dtype == THESEUS_VOCAB_BF16) launch<true>(p, pl, static_cast<uint8_t*>(workspace), stream);
        else launch<false>(p, pl, static_cast<uint8_t*>(workspace), stream);
    }
    return hipGetLastError() == hipSuccess ? THESEUS_WKV7_OK : THESEUS_WKV7_ERR_LAUNCH;
}

}  // extern "C"
