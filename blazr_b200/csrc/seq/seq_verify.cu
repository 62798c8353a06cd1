// seq_verify.cu -- drafted tokens against the target's probabilities, from given random numbers, and the token behind the accepted ones.
//
// Row r of entry e has logits z, the entry a temperature T, top_k and top_p:  w = exp((z - max z) / T), kept where z >= the k-th largest z and where the kept weights of
// strictly larger z are below top_p of their sum;  p = w / sum.  Draft x of row i is accepted when u_i q(x) < p(x).  The next token comes from max(p - q, 0) of the row that
// rejected (from p where that is nothing), or from the last row's p: the lowest one whose cumulated weight exceeds u times the sum.  T <= 0: p = 1 at the first maximum.
//
// What a row decides is compared with a random number, so that its sums are held in 64 bits.  The weights behind one comparison (a draft, the end of top_p) are f32, within 2^-21 of
// themselves; a draw is a comparison with 10^5 sums, and its weights are made in 64 bits, within 2^-34.
// Measured: 64 entries of 4 drafts, 128256 logits a row, 58 us (33.5 + 31; with draws of f32 weights 55, 28 of them; the logits' bytes alone 25, the draft's probabilities of a row an
// entry 5); one of 32000 logits 18.5, a chain of loads and of the clusters' barriers; 16 entries of 3 drafts with top_k and top_p 52 to 57 (thresholds 42 to 45).
// The floor is the logits' bytes: they are read once, in slices over the whole GPU (row_stats), with maximum, its place and sum left for every slice.  Then a cluster of eight
// CTAs an entry puts the slices together, finds the row that rejects and reads that one again, from L2, every warp a run of it (pick).
// top_k and top_p need a threshold a row before that (row_cut, a CTA a row, which it reads twice or three times from L2): counts, or masses (whole numbers of 2^-42: additions whose
// order does not matter, off by 2^-43 a token: 2^-26 of the largest weight for 128 k), of 2048 bins of equal width below the maximum show how far down the k-th logit lies, or where the mass passes the share; the logits down to there are sorted.
// Where those are too many (rows of equal logits, logits far apart), the threshold is selected by the bits of the ordered logits instead, eleven at a time.
#include <cfloat>
#include <cooperative_groups.h>

#include "seq_common.cuh"
#include "tc_split.cuh"

namespace b200seq {

namespace {

namespace cg = cooperative_groups;

constexpr int ERR_TOKEN = 16;             // error flag: a token id outside the vocabulary
constexpr int CLUSTER = 8;
constexpr int QUADS = 8;                  // 16-byte pieces of a slice of a row a thread has
constexpr int STATS = 256, PICK = 256, CUT = 1024;     // threads
constexpr int BINS = 2048, LIST = 2048;   // bins below the maximum; logits that are sorted
constexpr float MASS = 0x1p42f;           // masses as whole numbers: MAX_V weights of one fit 64 bits
constexpr int64_t MAX_V = (1 << 22) - 64;

struct Partial {      // of a slice of a row
    double sum;       // of exp((z - max) / T)
    float max;
    int at;           // lowest place of the maximum
};
struct Cut {          // of a row with top_k or top_p
    double total;     // of the weights that are kept, relative to the row's maximum
    float least;      // the smallest logit that is kept
    int on;
};

struct VerifyArgs {
    const float* x;
    int64_t ld;
    int R, V, B, slices;
    const int32_t *start, *drafts;
    const float *accept_u, *sample_u, *temp;
    const int32_t* top_k;
    const float *top_p, *q;
    int64_t ldq;
    int32_t *accepted, *tokens;
    Partial* part;     // [R][slices]
    Cut* cut;          // [R], with top_k or top_p
    int* err;
};

// four neighbouring logits at a 16-byte boundary of memory: quad k of a row holds the places 4 k - shift ...
__device__ __forceinline__ int quad_shift(const float* row) { return (int)((reinterpret_cast<uintptr_t>(row) >> 2) & 3); }
__device__ __forceinline__ float4 quad(const float* row, int i, int V, float none) {
    if (i >= 0 && i + 3 < V) return ld4(row + i);
    return make_float4(i >= 0 && i < V ? row[i] : none, i + 1 >= 0 && i + 1 < V ? row[i + 1] : none, i + 2 >= 0 && i + 2 < V ? row[i + 2] : none,
                       i + 3 >= 0 && i + 3 < V ? row[i + 3] : none);
}

// exp(d / T) = 2^(d c), c = log2(e) / T in two parts, so that the product is off by its own rounding alone
struct Heat {
    float hi, lo;
    __device__ __forceinline__ explicit Heat(float T) {
        const double c = fmin(1.4426950408889634 / (double)T, 3e38);
        hi = __double2float_rd(c), lo = (float)(c - (double)hi);      // (neither below zero: their products with d have one sign)
    }
    // weight of z under the maximum m: 1 at m, 0 at minus infinity; of a NaN, or under an infinite m, 0 (whoever sums looks for those)
    __device__ __forceinline__ float operator()(float z, float m) const {
        const float d = fmaxf(z - m, -FLT_MAX);
        return z == -INFINITY ? 0.f : tcsplit::ex2(fmaf(d, hi, d * lo));
    }
};

// The same weight to 2^-34 of itself: 2^u, u = (z - m) log2(e) / T, as 2^n 2^f with n whole and |f| <= 1/2, 2^f by the polynomial of the seventh degree that equals it at the Chebyshev
// nodes of that interval.  Logits below `least`, and those of weights below 2^-1000, have none.
struct FineHeat {
    double m, c;
    float lowest;
    __device__ __forceinline__ FineHeat(float T, float max, float least) {
        m = (double)max, c = 1.4426950408889634 / (double)T;
        lowest = fmaxf(fmaxf(__fsub_ru(max, __double2float_rd(1000.0 / c)), -FLT_MAX), least);
    }
    __device__ __forceinline__ double operator()(float z) const {
        const double d = (double)z - m, k = fma(d, c, 6755399441055744.0), f = fma(d, c, -(k - 6755399441055744.0));      // (1.5 2^52: the last digits are n)
        double p = 1.5303700711232177e-05;
        p = fma(p, f, 1.5469729214116396e-04), p = fma(p, f, 1.3333478473686084e-03), p = fma(p, f, 9.6180256133180427e-03), p = fma(p, f, 5.5504109063258658e-02);
        p = fma(p, f, 2.4022651213498092e-01), p = fma(p, f, 6.9314718055683244e-01), p = fma(p, f, 9.9999999995956179e-01);
        const int hi = __double2hiint(p) + (__double2loint(k) << 20);
        return z >= lowest ? __hiloint2double(hi, __double2loint(p)) : 0.0;
    }
};
// a finite number of normal size in 64 bits, by its bits (conversions go through a unit of a quarter of the rate); 0 as 2^-127, infinities and NaN as 2^128 or more
__device__ __forceinline__ double widened(float x) {
    const uint32_t b = __float_as_uint(x);
    return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + (896u << 20))), (int)(b << 29));
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// the entry that has a row (B: none); every thread of the block calls it
template <int THREADS>
__device__ __forceinline__ int entry_of(const VerifyArgs& a, int row) {
    int e = 0;
    for (int b0 = 0; b0 < a.B; b0 += THREADS) e += __syncthreads_count(b0 + (int)threadIdx.x < a.B && a.start[b0 + threadIdx.x + 1] <= row);
    return e;
}

// grid (slices, rows): 4 QUADS logits a thread, all asked for before anything else.  Small blocks, so that one's sums run beside another's loads (320 rows of 128256: blocks of 1024
// threads 64 us, of 256 40, with 32 logits a thread instead of 16 35; with the maximum's place looked up by those that have it and the weights two at a time 33.5: 4.9 TB/s, 13 instructions
// a logit for 21)
__global__ void __launch_bounds__(STATS) row_stats_kernel(const __grid_constant__ VerifyArgs a) {
    chain_enter();
    constexpr int THREADS = STATS, WARPS = THREADS / 32;
    __shared__ float wmax[WARPS];
    __shared__ unsigned wat[WARPS];
    __shared__ double wsum[WARPS];
    const int row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* x = a.x + row * a.ld;
    const int i0 = 4 * (blockIdx.x * QUADS * THREADS + threadIdx.x) - quad_shift(x);
    float4 v[QUADS];
#pragma unroll
    for (int k = 0; k < QUADS; ++k) v[k] = quad(x, i0 + 4 * k * THREADS, a.V, -INFINITY);
    const int e = entry_of<THREADS>(a, row);
    if (e >= a.B) return;
    const float T = a.temp[e];
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < QUADS; ++k) m = fmaxf(m, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
    const float wm = warp_max(m);
    if (lane == 0) wmax[warp] = wm;
    __syncthreads();
    float top = wmax[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, wmax[w]);
    unsigned at = 0x7fffffff;
    if (m == top && top > -INFINITY) {      // (few threads have it)
#pragma unroll
        for (int k = QUADS - 1; k >= 0; --k) {
            const int i = i0 + 4 * k * THREADS;
            at = v[k].x == top ? i : v[k].y == top ? i + 1 : v[k].z == top ? i + 2 : v[k].w == top ? i + 3 : at;
        }
    }
    const unsigned first = __reduce_min_sync(0xffffffffu, at);
    const Heat heat(T > 0.f ? T : 1.f);
    double sum = 0.0;      // (a slice of minus infinities: nothing)
    // the weights two at a time, with the roundings that heat() has; a sum that is no number has met one, or an infinity: heat() and a look at each.  (A difference beyond the type is
    // minus infinity here, the least number there: the same nothing, but for temperatures that make something of it.)
    const uint64_t off = tcsplit::pk(-top, -top), hi = tcsplit::pk(heat.hi, heat.hi), lo = tcsplit::pk(heat.lo, heat.lo);
    auto two = [&](float x, float y) {
        const uint64_t d = tcsplit::add2(tcsplit::pk(x, y), off);
        float a0, a1;
        tcsplit::upk(tcsplit::fma2(d, hi, tcsplit::mul2(d, lo)), a0, a1);
        return tcsplit::ex2(a0) + tcsplit::ex2(a1);
    };
#pragma unroll
    for (int k = 0; k < QUADS; ++k) sum += (double)(two(v[k].x, v[k].y) + two(v[k].z, v[k].w));
    if (!(sum >= 0.0) || T > 1e30f) {
        bool odd = false;
        sum = 0.0;
#pragma unroll
        for (int k = 0; k < QUADS; ++k) {
            odd |= v[k].x != v[k].x || v[k].y != v[k].y || v[k].z != v[k].z || v[k].w != v[k].w;
            if (top > -INFINITY) sum += (double)((heat(v[k].x, top) + heat(v[k].y, top)) + (heat(v[k].z, top) + heat(v[k].w, top)));
        }
        if (odd) sum = NAN;
    }
    sum = warp_sum(sum);
    if (lane == 0) wat[warp] = first, wsum[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned lo = wat[0];
        double s = wsum[0];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) lo = min(lo, wat[w]), s += wsum[w];
        a.part[(int64_t)row * a.slices + blockIdx.x] = Partial{s, top, (int)lo};
    }
}

// a row's maximum, its place, its sum; by one warp, the same in every lane.  sum is NaN (or the maximum infinite) where the row leaves no choice
struct Row {
    float max;
    int at;
    double sum;
    __device__ __forceinline__ bool none() const { return !(max > -INFINITY && max < INFINITY && sum > 0.0 && sum < INFINITY); }
};
__device__ __forceinline__ Row whole_row(const VerifyArgs& a, const Heat& heat, int row) {
    const Partial* p = a.part + (int64_t)row * a.slices;
    const int lane = threadIdx.x & 31;
    Row r{-INFINITY, 0x7fffffff, 0.0};
    for (int i = lane; i < a.slices; i += 32) r.max = fmaxf(r.max, p[i].max);
    r.max = warp_max(r.max);
    unsigned at = 0x7fffffff;
    for (int i = lane; i < a.slices; i += 32) {
        const Partial s = p[i];
        if (s.max == r.max) at = min(at, (unsigned)s.at);
        r.sum += s.sum * (double)heat(s.max, r.max);      // (0 or NaN stay what they are)
    }
    r.at = (int)__reduce_min_sync(0xffffffffu, at);
    r.sum = warp_sum(r.sum);
    return r;
}

// logits as whole numbers of the same order (-0 as 0)
__device__ __forceinline__ uint32_t order_key(float z) {
    const uint32_t b = __float_as_uint(z + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

// the sum of a number of every thread, for all; sh: 33 words
template <class N>
__device__ __forceinline__ N block_total(N v, N* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();                                       // (sh may still be read)
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// what lies before a thread's number, in the order of the threads (from the last on: FROM_TOP); sh: 32 words
template <class N, bool FROM_TOP>
__device__ __forceinline__ N block_before(N own, N* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    N s = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const N y = FROM_TOP ? __shfl_down_sync(0xffffffffu, s, o) : __shfl_up_sync(0xffffffffu, s, o);
        if (FROM_TOP ? lane + o < 32 : lane >= o) s += y;
    }
    __syncthreads();                                       // (sh may still be read)
    if (lane == (FROM_TOP ? 0 : 31)) sh[warp] = s;
    __syncthreads();
    N w = sh[lane], all = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const N y = FROM_TOP ? __shfl_down_sync(0xffffffffu, all, o) : __shfl_up_sync(0xffffffffu, all, o);
        if (FROM_TOP ? lane + o < 32 : lane >= o) all += y;
    }
    return s - own + __shfl_sync(0xffffffffu, all - w, warp);
}

// Of 2048 bins, bins 2 t and 2 t + 1 in thread t, the one in which what is added up (from the last bin on: FROM_TOP) passes `want`, and what comes before it; for all threads
template <bool FROM_TOP>
__device__ __forceinline__ int find_bin(unsigned long long b0, unsigned long long b1, unsigned long long want, unsigned long long& before, unsigned long long* sh) {
    const unsigned long long first = FROM_TOP ? b1 : b0, second = FROM_TOP ? b0 : b1, s = block_before<unsigned long long, FROM_TOP>(b0 + b1, sh);
    const int t = 2 * threadIdx.x;
    if (s < want && s + first >= want) sh[32] = t + (FROM_TOP ? 1 : 0), sh[33] = s;
    if (s + first < want && s + first + second >= want) sh[32] = t + (FROM_TOP ? 0 : 1), sh[33] = s + first;
    __syncthreads();
    before = sh[33];
    return (int)sh[32];
}

// a row's logits, every thread its share of them
template <class F>
__device__ __forceinline__ void each_logit(const float* x, int V, F f) {
    const int shift = quad_shift(x), quads = (V + shift + 3) / 4;
#pragma unroll 2
    for (int k = threadIdx.x; k < quads; k += CUT) {
        const int i = 4 * k - shift;
        if (i >= 0 && i + 3 < V) {
            const float4 v = ld4(x + i);
            f(v.x), f(v.y), f(v.z), f(v.w);
        } else {
            for (int j = max(i, 0); j < min(i + 4, V); ++j) f(x[j]);
        }
    }
}

// The smallest ordered logit that is kept, by its bits.  h: a table of 2048.
__device__ __noinline__ uint32_t slow_cut(const float* x, int V, float top, const Heat heat, int k, bool by_count, bool by_mass, float share, unsigned long long* h, unsigned long long* sh) {
    const int tid = threadIdx.x;
    uint32_t least = 0;                                     // keys from here on are kept
    for (int pass = 0; pass < 2; ++pass) {
        if (pass == 0 ? !by_count : !by_mass) continue;
        uint32_t prefix = 0;
        unsigned long long want = (unsigned long long)k;
        for (int level = 0; level < 3; ++level) {
            const int bits = level < 2 ? 11 : 10, shift = level == 0 ? 21 : level == 1 ? 10 : 0;
            __syncthreads();
            h[tid] = h[tid + 1024] = 0;
            __syncthreads();
            each_logit(x, V, [&](float z) {
                const uint32_t key = order_key(z);
                if (key < least || (level > 0 && (key >> (shift + bits)) != prefix)) return;
                unsigned long long add = 1;
                if (pass == 1) add = __float2ull_rn(heat(z, top) * MASS);
                if (add) atomicAdd(h + ((key >> shift) & ((1u << bits) - 1)), add);
            });
            __syncthreads();
            const unsigned long long b0 = h[2 * tid], b1 = h[2 * tid + 1];
            if (pass == 1 && level == 0) {
                const double t = ceil((double)share * (double)block_total(b0 + b1, sh));
                want = t >= 1.0 ? (unsigned long long)t : 1ull;
            }
            unsigned long long over;
            const int bin = find_bin<true>(b0, b1, want, over, sh);
            want -= over;
            prefix = level == 0 ? (uint32_t)bin : (prefix << bits) | (uint32_t)bin;
        }
        least = prefix;
    }
    return least;
}

// grid (rows)
__global__ void __launch_bounds__(CUT, 1) row_cut_kernel(const __grid_constant__ VerifyArgs a) {
    chain_enter();
    __shared__ __align__(16) unsigned h32[4 * BINS];        // bins: counts, masses in three parts; or the slow way's table
    __shared__ unsigned long long sh[34];
    __shared__ unsigned list[LIST], many, next, cut_key;
    __shared__ Row row_sh;
    const int row = blockIdx.x, tid = threadIdx.x;
    const int e = entry_of<CUT>(a, row);
    if (e >= a.B) return;
    const int k = a.top_k ? a.top_k[e] : 0;
    const float share = a.top_p ? a.top_p[e] : 1.f, T = a.temp[e];
    bool by_count = k > 0 && k < a.V;
    const bool by_mass = share < 1.f;
    if (!(T > 0.f) || !(by_count || by_mass)) {
        if (tid == 0) a.cut[row] = Cut{0.0, 0.f, 0};
        return;
    }
    const Heat heat(T);
    for (int i = tid; i < 4 * BINS; i += CUT) h32[i] = 0;
    if (tid < 32) {
        const Row r = whole_row(a, heat, row);
        if (tid == 0) row_sh = r, many = 0, next = 0, cut_key = 0;
    }
    __syncthreads();
    const Row r = row_sh;
    if (r.none()) {
        if (tid == 0) a.cut[row] = Cut{0.0, 0.f, 0};
        return;
    }
    const float* x = a.x + row * a.ld;
    const float width = (float)BINS / (32.f * fmaxf(T, 1.f));
    bool masses_only = false;                               // (the counts are there)
    // (numbers made whole by adding 2^23: conversions, like the exponential, go through a unit of a quarter of the rate)
    auto bin_of = [&](float z) { return (int)(__float_as_uint(fminf((r.max - z) * width, (float)(BINS - 1)) + 8388608.f) & (2 * BINS - 1)); };
    // ---- counts, and masses where they are needed: with top_k, of few logits later ----
    int finite = 0;
    for (bool again = true; again;) {
        each_logit(x, a.V, [&](float z) {
            const int b = bin_of(z);
            finite += z > -INFINITY;
            if (b == BINS - 1) return;                      // (the last bin has what the others have not; a weight in it is below 2^-46)
            if (by_count || !masses_only) atomicAdd(h32 + b, 1u);
            if (!by_count) {
                const float w = heat(z, r.max) * 65536.f, c = w + 8388608.f;
                const unsigned whole = __float_as_uint(c) & 0x1ffffu;
                const float x1 = (w - (c - 8388608.f)) * 65536.f, c1 = x1 + 12582912.f;
                const int part = (int)(__float_as_uint(c1) - 0x4B400000u);      // (-32768 .. 32768: 32768 of either fit 32 bits)
                const int low = (int)(__float_as_uint((x1 - (c1 - 12582912.f)) * 1024.f + 12582912.f) - 0x4B400000u);
                if (whole) atomicAdd(h32 + BINS + b, whole);
                if (part) atomicAdd(reinterpret_cast<int*>(h32) + 2 * BINS + b, part);
                if (low) atomicAdd(reinterpret_cast<int*>(h32) + 3 * BINS + b, low);
            }
        });
        again = false;
        if (by_count && !masses_only && (unsigned long long)k >= block_total((unsigned long long)finite, sh)) {      // (all but minus infinities are kept)
            by_count = false;
            if (!by_mass) {
                if (tid == 0) a.cut[row] = Cut{0.0, 0.f, 0};
                return;
            }
            again = masses_only = true;
        }
    }
    __syncthreads();
    const int b0 = 2 * tid, b1 = b0 + 1;
    unsigned long long c0 = h32[b0], c1 = h32[b1];
    if (c0 > 32768 || c1 > 32768) many = 1;
    const unsigned long long in_all = block_total(c0 + c1, sh);
    if (b1 == BINS - 1) c1 = a.V - in_all;
    unsigned long long want, before, all_mass = 0;
    int b;
    if (by_count) {
        want = (unsigned long long)k;
        b = find_bin<false>(c0, c1, want, before, sh);
    } else {
        auto mass = [&](int i) {      // (never below zero: a sum of numbers that are not)
            return ((unsigned long long)h32[BINS + i] << 26) + (unsigned long long)((long long)(int)h32[2 * BINS + i] * 1024 + (int)h32[3 * BINS + i]);
        };
        const unsigned long long m0 = mass(b0), m1 = mass(b1);
        all_mass = block_total(m0 + m1, sh);
        const double t = ceil((double)share * (double)all_mass);
        want = t >= 1.0 ? (unsigned long long)t : 1ull;
        b = find_bin<false>(m0, m1, want, before, sh);
    }
    // the logits of this bin and of those before it, sorted; or, where top_p is all there is, of this bin alone
    unsigned n = (unsigned)min(block_total((b0 <= b ? c0 : 0ull) + (b1 <= b ? c1 : 0ull), sh), (unsigned long long)LIST + 1);
    const bool alone = n > LIST / 4 && !by_count;           // (a pass over the row takes less than sorting so many)
    if (alone) n = (unsigned)min(block_total((b0 == b ? c0 : 0ull) + (b1 == b ? c1 : 0ull), sh), (unsigned long long)LIST + 1);
    uint32_t least;
    double total = 0.0;
    if (n > LIST || many) {
        __syncthreads();
        least = slow_cut(x, a.V, r.max, heat, k, by_count, by_mass, share, reinterpret_cast<unsigned long long*>(h32), sh);
        each_logit(x, a.V, [&](float z) {
            if (order_key(z) >= least) total += (double)heat(z, r.max);
        });
    } else {
        each_logit(x, a.V, [&](float z) {
            const int at = bin_of(z);
            if (alone ? at == b : at <= b) list[atomicAdd(&next, 1u)] = order_key(z);
        });
        __syncthreads();
        int size = 32;
        while (size < (int)n) size <<= 1;
        for (int i = (int)n + tid; i < size; i += CUT) list[i] = 0;
        __syncthreads();
        for (int run = 2; run <= size; run <<= 1)           // bitonic, the largest first
            for (int step = run >> 1; step > 0; step >>= 1) {
                if (tid < size / 2) {
                    const int at = ((tid & ~(step - 1)) << 1) | (tid & (step - 1)), to = at + step;
                    const unsigned u = list[at], v = list[to];
                    if ((u < v) == ((at & run) == 0)) list[at] = v, list[to] = u;
                }
                // (a warp has 64 neighbours to itself: shorter steps stay within them)
                if (step > 32 || (step == 1 && run >= 64)) __syncthreads();
                else __syncwarp();
            }
        __syncthreads();
        least = by_count ? list[k - 1] : 0;
        double w[2];                                        // two neighbours a thread, of those that top_k leaves
        uint32_t key[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            key[i] = 2 * tid + i < size ? list[2 * tid + i] : 0;
            w[i] = key[i] > 0 && key[i] >= least ? (double)heat(key_value(key[i]), r.max) : 0.0;
        }
        double* const d = reinterpret_cast<double*>(sh);
        if (by_mass) {
            const double all = by_count ? block_total(w[0] + w[1], d) : (double)all_mass * (1.0 / MASS), goal = (double)share * all;
            const double up = block_before<double, false>(w[0] + w[1], d) + (alone ? (double)before * (1.0 / MASS) : 0.0);
            // the last one with less than the goal before it (the largest always)
            uint32_t last = tid == 0 ? key[0] : 0xffffffffu;
            if (w[0] > 0.0 && up < goal) last = key[0];
            if (w[1] > 0.0 && up + w[0] < goal) last = key[1];
            last = __reduce_min_sync(0xffffffffu, last);
            if ((tid & 31) == 0 && last != 0xffffffffu) atomicMax(&cut_key, ~last);
            __syncthreads();
            least = max(least, ~cut_key);
        }
        total = (key[0] >= least ? w[0] : 0.0) + (key[1] >= least ? w[1] : 0.0);
        if (alone) {
            total = 0.0;
            each_logit(x, a.V, [&](float z) {
                if (order_key(z) >= least) total += (double)heat(z, r.max);
            });
        }
    }
    total = block_total(total, reinterpret_cast<double*>(sh));
    if (tid == 0) a.cut[row] = Cut{total, key_value(least), 1};
}

// what a warp or a block has of a row: the weights to draw from, all weights, and the draft's probabilities where weights are left
struct Share {
    double draw, all;
    float off;
    __device__ __forceinline__ void add(const Share& o) { draw += o.draw, all += o.all, off += o.off; }
};

// grid: a cluster an entry
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(PICK) pick_kernel(const __grid_constant__ VerifyArgs a) {
    chain_enter();
    constexpr int WARPS = PICK / 32, ROWS = 32, AHEAD = 4;
    __shared__ double scan[PICK], warp_part[WARPS];
    __shared__ Share warp_share[WARPS], cta_share;
    __shared__ int first_bad, found, last_some;
    __shared__ Row rows_sh[ROWS], row_sh;
    cg::cluster_group cl = cg::this_cluster();
    const int e = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int s0 = a.start[e], s1 = a.start[e + 1];
    const float T = a.temp[e], u_e = a.sample_u[e];
    if (s0 < 0 || s1 < s0 || s1 > a.R || s0 == s1) {        // no rows, or no list of rows (the whole cluster alike)
        if (rank == 0 && tid == 0) {
            a.accepted[e] = 0;
            if (s0 != s1) atomicOr(a.err, ERR_TOKEN);
        }
        return;
    }
    const int n = s1 - s0 - 1;
    const bool greedy = !(T > 0.f);
    const Heat heat(greedy ? 1.f : T);
    if (tid == 0) first_bad = n;
    __syncthreads();
    for (int i = warp; i <= n; i += WARPS) {
        const int row = s0 + i, x = i < n ? a.drafts[row] : 0;
        const bool in = x >= 0 && x < a.V;
        float z = 0.f, u = 0.f, q = 1.f;
        if (i < n && in && !greedy) {      // (asked for beside the slices)
            z = a.x[row * a.ld + x], u = a.accept_u[row];
            if (a.q) q = a.q[row * a.ldq + x];
        }
        const Row r = whole_row(a, heat, row);
        if (lane == 0) {
            if (i < ROWS) rows_sh[i] = r;
            bool fine = false;
            if (!in) atomicOr(a.err, ERR_TOKEN);
            else if (!r.none()) {
                if (greedy) fine = x == r.at;
                else {
                    double w = (double)heat(z, r.max), sum = r.sum;
                    if (a.cut && a.cut[row].on) sum = a.cut[row].total, w = z >= a.cut[row].least ? w : 0.0;
                    fine = (double)u * (double)q < w / sum;
                }
            }
            if (!fine && i < n) atomicMin(&first_bad, i);
        }
    }
    __syncthreads();
    const int acc = first_bad, row = s0 + acc;
    if (acc >= ROWS && warp == 0) {
        const Row r = whole_row(a, heat, row);
        if (lane == 0) row_sh = r;
    }
    if (rank == 0) {
        for (int i = tid; i <= n; i += PICK)
            if (i != acc) a.tokens[s0 + i] = i < acc ? a.drafts[s0 + i] : -1;
        if (tid == 0) a.accepted[e] = acc;
    }
    if (acc >= ROWS) __syncthreads();
    const Row r = acc < ROWS ? rows_sh[acc] : row_sh;
    if (r.none() || greedy) {
        if (rank == 0 && tid == 0) a.tokens[row] = r.none() ? -1 : r.at;
        return;
    }
    float least = -INFINITY;
    double about = r.sum;                                   // the row's sum, to the digits of 32-bit weights
    if (a.cut && a.cut[row].on) about = a.cut[row].total, least = a.cut[row].least;
    const float* x = a.x + row * a.ld;
    const float* q = a.q && acc < n ? a.q + row * a.ldq : nullptr;
    const int certain = acc < n && !q ? a.drafts[row] : -1, shift = quad_shift(x);
    const bool aligned_q = q && (quad_shift(q) == shift);
    // Weights in 64 bits: which of 10^5 sums is the first beyond the target is known only to their own digits (in 32 bits one draw in 10^4 was the neighbour's).  Drawn from is what
    // w has more than S q, S the sum of all w.  That is known only behind the walk over the row, which takes `about` for S: where weights are left, sums of q tell what that changes.
    const FineHeat weight(T, r.max, least);
    auto load = [&](int k, float4& z, float4& qv) {
        const int i = 4 * k - shift;
        z = quad(x, i, a.V, -INFINITY), qv = make_float4(0.f, 0.f, 0.f, 0.f);
        if (q) {
            if (aligned_q) qv = quad(q, i, a.V, 0.f);
            else qv = make_float4(i >= 0 && i < a.V ? q[i] : 0.f, i + 1 >= 0 && i + 1 < a.V ? q[i + 1] : 0.f, i + 2 >= 0 && i + 2 < a.V ? q[i + 2] : 0.f,
                                  i + 3 >= 0 && i + 3 < a.V ? q[i + 3] : 0.f);
        }
    };
    // the four weights of a lane; false: the whole warp has none
    auto weights = [&](const float4& z, double (&w)[4]) {
        const bool some = __any_sync(0xffffffffu, fmaxf(fmaxf(z.x, z.y), fmaxf(z.z, z.w)) >= weight.lowest);
        if (some) w[0] = weight(z.x), w[1] = weight(z.y), w[2] = weight(z.z), w[3] = weight(z.w);
        return some;
    };
    auto left = [&](double w, float qv, double all) {      // (a q that is no number takes all)
        if (!q) return w;
        const double l = fma(-all, widened(qv), w);
        return __double2hiint(l) < 0 ? 0.0 : l;
    };
    // every warp a run of neighbouring quads, every lane its sums, AHEAD quads asked for at a time (64 entries with drafts' probabilities, in all: one 61.8 us, two 60.9, four 58.0)
    const int quads = (a.V + shift + 3) / 4, run = ((quads + CLUSTER * WARPS - 1) / (CLUSTER * WARPS) + 31) & ~31;
    Share mine{0.0, 0.0, 0.f};
    const int k0 = (rank * WARPS + warp) * run;
    const int k1 = min(k0 + run, (quads + 31) & ~31);
    for (int kk = k0 + lane; kk < k1; kk += 32 * AHEAD) {
        float4 z[AHEAD], qv[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) load(kk + 32 * u < k1 ? kk + 32 * u : quads, z[u], qv[u]);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            double w[4];
            if (!weights(z[u], w)) continue;
            const float qs[4] = {qv[u].x, qv[u].y, qv[u].z, qv[u].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mine.all += w[j];
                const double l = 4 * (kk + 32 * u) - shift + j == certain ? 0.0 : left(w[j], qs[j], about);
                mine.draw += l;
                if (q && __double2hiint(l) > 0) mine.off += qs[j];
            }
        }
    }
    mine.draw = warp_sum(mine.draw), mine.all = warp_sum(mine.all);
    if (q) mine.off = warp_sum(mine.off);
    if (lane == 0) warp_share[warp] = mine;
    __syncthreads();
    if (tid == 0) {
        Share y = warp_share[0];
        for (int k = 1; k < WARPS; ++k) y.add(warp_share[k]);
        cta_share = y;
    }
    cl.sync();
    Share row_share{0.0, 0.0, 0.f}, share[CLUSTER];
#pragma unroll
    for (int k = 0; k < CLUSTER; ++k) share[k] = *cl.map_shared_rank(&cta_share, k), row_share.add(share[k]);
    const double more = q ? row_share.all - about : 0.0;
    const bool rest = row_share.draw - more * (double)row_share.off > 0.0;      // (else nothing is left of the draft's excess: the target's own probabilities)
    auto drawn = [&](const Share& y) { return rest ? y.draw - more * (double)y.off : y.all; };
    const double target = (double)u_e * drawn(row_share);
    double before = 0.0, base = 0.0;
    bool passed = false;
    int owner = -1;                                         // the CTA in whose share the sum passes the target (rounding: the last that has any)
#pragma unroll
    for (int k = 0; k < CLUSTER; ++k) {
        const double y = drawn(share[k]);
        if (y > 0.0 && !passed) owner = k, base = before, passed = before + y > target;
        before += y;
    }
    if (rank == owner) {
        int of = 0;
        before = base;
        for (int k = 0; k < WARPS; ++k) {
            const double y = drawn(warp_share[k]);
            if (y > 0.0) {
                of = k, base = before;
                if (before + y > target) break;
            }
            before += y;
        }
        if (tid == 0) found = 0x7fffffff, last_some = -1;
        __syncthreads();
        // that warp's run, by the block: a tile of its quads at a time
        const int from = (rank * WARPS + of) * run, to = min(from + run, quads);
        for (int t = from; t < to; t += PICK) {
            double w[4] = {0.0, 0.0, 0.0, 0.0};
            float4 z, qv;
            const int k = t + tid;
            load(k < to ? k : quads, z, qv);                // (behind the last quad: minus infinities)
            weights(z, w);
            const float qs[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (rest) w[j] = 4 * k - shift + j == certain ? 0.0 : left(w[j], qs[j], row_share.all);
            const double own = (w[0] + w[1]) + (w[2] + w[3]);
            double s = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += y;
            }
            if (lane == 31) warp_part[warp] = s;
            __syncthreads();
            for (int v = 0; v < warp; ++v) s += warp_part[v];
            scan[tid] = s;
            __syncthreads();
            double cum = base + (tid ? scan[tid - 1] : 0.0);
            if (own > 0.0) {
                int last = -1;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    cum += w[j];
                    if (w[j] > 0.0) {
                        last = 4 * k - shift + j;
                        if (cum > target) {
                            atomicMin(&found, last);
                            break;
                        }
                    }
                }
                atomicMax(&last_some, last);
            }
            base += scan[PICK - 1];
            __syncthreads();
            if (found != 0x7fffffff) break;
        }
        if (tid == 0) a.tokens[row] = found != 0x7fffffff ? found : last_some;
    }
    cl.sync();                                              // nobody's sums go while they are read
}

int slices_of(int V) { return (V + 3 + 4 * QUADS * STATS - 1) / (4 * QUADS * STATS); }

}  // namespace

}  // namespace b200seq

using namespace b200seq;

extern "C" {

size_t b200seq_verify_scratch_bytes(int R, int V, int ruled) {
    if (R < 1 || V < 1 || V > MAX_V) return 0;
    return (size_t)R * slices_of(V) * sizeof(Partial) + (ruled ? (size_t)R * sizeof(Cut) : 0);
}

int b200seq_verify_drafts(const float* logits, int64_t ld, int R, int V, const int32_t* start, int B, const int32_t* drafts, const float* accept_u, const float* sample_u,
                          const float* temperature, const int32_t* top_k, const float* top_p, const float* draft_probs, int64_t ldq, int32_t* accepted, int32_t* tokens,
                          void* scratch, size_t scratch_bytes, void* stream) {
    if (R < 0 || B < 0 || V < 1 || (B > 0 && (!start || !sample_u || !temperature || !accepted)) || (R > 0 && B > 0 && (!logits || !drafts || !accept_u || !tokens || !scratch)))
        return fail(B200SEQ_ERR_INVALID_ARG, "verify_drafts: bad sizes or null arrays");
    if (R > 65535 || B > (1 << 24)) return fail(B200SEQ_ERR_UNSUPPORTED, "verify_drafts: up to 65535 rows");
    if (V > MAX_V) return fail(B200SEQ_ERR_UNSUPPORTED, "verify_drafts: up to %lld tokens in a vocabulary", (long long)MAX_V);
    if (R > 1 && (ld < V || (draft_probs && ldq < V))) return fail(B200SEQ_ERR_INVALID_ARG, "verify_drafts: row strides below a row's length");
    const bool ruled = top_k || top_p;
    if (R > 0 && B > 0 && (scratch_bytes < b200seq_verify_scratch_bytes(R, V, ruled) || (reinterpret_cast<uintptr_t>(scratch) & 15)))
        return fail(B200SEQ_ERR_INVALID_ARG, "verify_drafts: the work area is too small or not on a 16-byte boundary");
    if (B == 0) return 0;
    if (R > 0 && tokens < drafts + R && drafts < tokens + R) return fail(B200SEQ_ERR_INVALID_ARG, "verify_drafts: tokens and drafts share memory");      // (read by other blocks than write them)
    VerifyArgs a{logits, ld, R, V, B, 0, start, drafts, accept_u, sample_u, temperature, top_k, top_p, draft_probs, ldq, accepted, tokens, (Partial*)scratch, nullptr, error_flag_dev()};
    a.slices = slices_of(V);
    if (ruled) a.cut = reinterpret_cast<Cut*>(a.part + (size_t)R * a.slices);
    const cudaStream_t cs = (cudaStream_t)stream;
    if (R > 0) {
        launch_chained(row_stats_kernel, dim3(a.slices, R), STATS, 0, cs, a);
        SEQ_LAUNCH_CHECK("verify_drafts");
        if (ruled) {
            launch_chained(row_cut_kernel, dim3(R), CUT, 0, cs, a);
            SEQ_LAUNCH_CHECK("verify_drafts");
        }
    }
    launch_chained(pick_kernel, dim3(CLUSTER * B), PICK, 0, cs, a);
    SEQ_LAUNCH_CHECK("verify_drafts");
    return 0;
}

}  // extern "C"
