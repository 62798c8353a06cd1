// seq_verify.cu -- drafted tokens against the target's probabilities, from given random numbers, and the token behind the accepted ones.
//
// Row r of entry e has logits z, the entry a temperature T, top_k and top_p:  w = exp((z - max z) / T), kept where z >= the k-th largest z and where the kept weights of
// strictly larger z are below top_p of their sum;  p = w / sum.  Draft x of row i is accepted when u_i q(x) < p(x).  The next token comes from max(p - q, 0) of the row that
// rejected (from p where that is nothing), or from the last row's p: the lowest one whose cumulated weight exceeds u times the sum.  T <= 0: p = 1 at the first maximum.
//
// What a row decides is compared with a random number, so that its sums are held in 64 bits (weights are f32, within 2^-21 of themselves; sums of four of them, then f64).
// The floor is the logits' bytes: they are read once, in slices over the whole GPU (row_stats), with maximum, its place and sum left for every slice.  Then a cluster of eight
// CTAs an entry puts the slices together, finds the row that rejects and reads that one again, from L2 (pick).  top_k and top_p need a threshold a row before that: a cluster a
// row selects it by the bits of the ordered logits, eleven at a time, by counts, then by masses in whole numbers of 2^-31 (row_cut): additions whose order does not matter.
#include <cooperative_groups.h>

#include "seq_common.cuh"
#include "tc_split.cuh"

namespace b200seq {

namespace {

namespace cg = cooperative_groups;

constexpr int ERR_TOKEN = 16;             // error flag: a token id outside the vocabulary
constexpr int CLUSTER = 8;
constexpr int PICK = 512, CUT = 1024;     // threads
constexpr int MAX_TILES = 512;            // tiles of 4 * PICK logits of one CTA's share
constexpr int64_t MAX_V = (int64_t)CLUSTER * MAX_TILES * 4 * PICK - 64;

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
        hi = (float)c, lo = (float)(c - (double)hi);
    }
    // weight of z under the maximum m; NaN where either is no number
    __device__ __forceinline__ float operator()(float z, float m) const {
        if (z == m && m > -INFINITY && m < INFINITY) return 1.f;
        if (z == -INFINITY) return 0.f;
        const float d = z - m;
        return tcsplit::ex2(fmaf(d, hi, d * lo));
    }
};

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

// grid (slices, rows): 16 logits a thread, all asked for before anything else
template <int THREADS>
__global__ void __launch_bounds__(THREADS) row_stats_kernel(const __grid_constant__ VerifyArgs a) {
    chain_enter();
    constexpr int WARPS = THREADS / 32;
    __shared__ float wmax[WARPS];
    __shared__ unsigned wat[WARPS];
    __shared__ double wsum[WARPS];
    const int row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* x = a.x + row * a.ld;
    const int i0 = 4 * (blockIdx.x * 4 * THREADS + threadIdx.x) - quad_shift(x);
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = quad(x, i0 + 4 * k * THREADS, a.V, -INFINITY);
    const int e = entry_of<THREADS>(a, row);
    if (e >= a.B) return;
    const float T = a.temp[e];
    float m = -INFINITY;
    int at = 0x7fffffff;
    bool odd = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float z[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (z[j] > m) m = z[j], at = i0 + 4 * k * THREADS + j;
            odd |= z[j] != z[j];
        }
    }
    const float wm = warp_max(m);
    if (lane == 0) wmax[warp] = wm;
    __syncthreads();
    float top = wmax[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, wmax[w]);
    const unsigned first = __reduce_min_sync(0xffffffffu, m == top && top > -INFINITY ? (unsigned)at : 0x7fffffffu);
    const Heat heat(T > 0.f ? T : 1.f);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) sum += (double)((heat(v[k].x, top) + heat(v[k].y, top)) + (heat(v[k].z, top) + heat(v[k].w, top)));
    if (odd) sum = NAN;
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
        r.sum += s.sum == 0.0 ? 0.0 : s.sum * (double)heat(s.max, r.max);
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

// The bin of an array of 2048 (two neighbours a thread) in which what lies above, added up from the top, passes `want`: the lowest bin with fewer than `want` above it and
// something in it.  Every thread gets the bin and what lies above it.  sh: 34 words.
__device__ __forceinline__ int find_bin(unsigned long long lo, unsigned long long hi, unsigned long long want, unsigned long long& above, unsigned long long* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long s = lo + hi;                        // bins 2 t, 2 t + 1: from this thread's to the warp's last
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_down_sync(0xffffffffu, s, o);
        if (lane + o < 32) s += y;
    }
    __syncthreads();                                       // (sh may still be read)
    if (lane == 0) sh[warp] = s;
    __syncthreads();
    for (int w = warp + 1; w < CUT / 32; ++w) s += sh[w];
    const unsigned long long over = s - lo - hi;           // above both bins
    if (hi > 0 && over < want && over + hi >= want) sh[32] = 2 * threadIdx.x + 1, sh[33] = over;
    if (lo > 0 && over + hi < want && over + hi + lo >= want) sh[32] = 2 * threadIdx.x, sh[33] = over + hi;
    __syncthreads();
    above = sh[33];
    return (int)sh[32];
}

// grid (8 rows' worth of clusters): a cluster a row
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(CUT) row_cut_kernel(const __grid_constant__ VerifyArgs a) {
    chain_enter();
    __shared__ unsigned long long hist[2][2048];
    __shared__ unsigned long long sh[34];
    __shared__ Row row_sh;
    cg::cluster_group cl = cg::this_cluster();
    const int row = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER, tid = threadIdx.x;
    const int e = entry_of<CUT>(a, row);
    if (e >= a.B) return;                                   // (the whole cluster alike, here and below)
    const int k = a.top_k ? a.top_k[e] : 0;
    const float share = a.top_p ? a.top_p[e] : 1.f, T = a.temp[e];
    const bool by_count = k > 0 && k < a.V, by_mass = share < 1.f;
    if (!(T > 0.f) || !(by_count || by_mass)) {
        if (rank == 0 && tid == 0) a.cut[row] = Cut{0.0, 0.f, 0};
        return;
    }
    const Heat heat(T);
    if (tid < 32) {
        const Row r = whole_row(a, heat, row);
        if (tid == 0) row_sh = r;
    }
    __syncthreads();
    const Row r = row_sh;
    if (r.none()) {
        if (rank == 0 && tid == 0) a.cut[row] = Cut{0.0, 0.f, 0};
        return;
    }
    const int share_v = (a.V + CLUSTER - 1) / CLUSTER, lo = min(a.V, rank * share_v), hi = min(a.V, lo + share_v);
    const float* x = a.x + row * a.ld;
    int buf = 0;
    uint32_t least = 0;                                     // keys from here on are kept
    double total = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        if (pass == 0 ? !by_count : !by_mass) continue;
        uint32_t prefix = 0;
        unsigned long long want = (unsigned long long)k, above = 0;
        for (int level = 0; level < 3; ++level) {
            const int bits = level < 2 ? 11 : 10, shift = level == 0 ? 21 : level == 1 ? 10 : 0;
            unsigned long long* h = hist[buf];
            h[tid] = h[tid + 1024] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += CUT) {
                const float z = x[i];
                const uint32_t key = order_key(z);
                if (key < least || (level > 0 && (key >> (shift + bits)) != prefix)) continue;
                unsigned long long add = 1;
                if (pass == 1) add = (unsigned long long)__float2uint_rn(heat(z, r.max) * 0x1p31f);
                if (add) atomicAdd(h + ((key >> shift) & ((1u << bits) - 1)), add);
            }
            cl.sync();
            unsigned long long b0 = 0, b1 = 0;              // every CTA adds all eight up for itself: whole numbers, the same sums everywhere
            for (int c = 0; c < CLUSTER; ++c) {
                const unsigned long long* o = cl.map_shared_rank(h, c);
                b0 += o[2 * tid], b1 += o[2 * tid + 1];
            }
            if (pass == 1 && level == 0) {
                unsigned long long all = b0 + b1;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
                __syncthreads();
                if ((tid & 31) == 0) sh[tid >> 5] = all;
                __syncthreads();
                all = 0;
                for (int w = 0; w < CUT / 32; ++w) all += sh[w];
                const double t = ceil((double)share * (double)all);
                want = t >= 1.0 ? (unsigned long long)t : 1ull;
            }
            unsigned long long over;
            const int bin = find_bin(b0, b1, want, over, sh);
            want -= over, above += over;
            prefix = level == 0 ? (uint32_t)bin : (prefix << bits) | (uint32_t)bin;
            if (pass == 1 && level == 2) {                  // (the bin is one value: what it holds is kept)
                __syncthreads();
                if (tid == bin >> 1) sh[32] = above + (bin & 1 ? b1 : b0);
                __syncthreads();
                total = (double)sh[32] * 0x1p-31;
            }
            buf ^= 1;
        }
        least = prefix;
    }
    // (without top_p: the sum of the k largest, in the order of the places)
    if (!by_mass) {
        double s = 0.0;
        for (int i = lo + tid; i < hi; i += CUT)
            if (order_key(x[i]) >= least) s += (double)heat(x[i], r.max);
        s = warp_sum(s);
        double* d = reinterpret_cast<double*>(sh);
        __syncthreads();
        if ((tid & 31) == 0) d[tid >> 5] = s;
        __syncthreads();
        if (tid == 0) {
            s = 0.0;
            for (int w = 0; w < CUT / 32; ++w) s += d[w];
            d[32] = s;
        }
        cl.sync();
        if (rank == 0 && tid == 0)
            for (int c = 0; c < CLUSTER; ++c) total += *cl.map_shared_rank(d + 32, c);
    }
    if (rank == 0 && tid == 0) a.cut[row] = Cut{total, key_value(least), 1};
    cl.sync();                                              // nobody's tables go while they are read
}

// grid: a cluster an entry
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(PICK) pick_kernel(const __grid_constant__ VerifyArgs a) {
    chain_enter();
    __shared__ double tile_sum[MAX_TILES], scan[PICK], warp_part[PICK / 32], cta_sum;
    __shared__ int first_bad, found, last_some;
    __shared__ Row row_sh;
    cg::cluster_group cl = cg::this_cluster();
    const int e = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int s0 = a.start[e], s1 = a.start[e + 1];
    if (s0 < 0 || s1 < s0 || s1 > a.R || s0 == s1) {        // no rows, or no list of rows (the whole cluster alike)
        if (rank == 0 && tid == 0) {
            a.accepted[e] = 0;
            if (s0 != s1) atomicOr(a.err, ERR_TOKEN);
        }
        return;
    }
    const int n = s1 - s0 - 1;
    const float T = a.temp[e];
    const bool greedy = !(T > 0.f);
    const Heat heat(greedy ? 1.f : T);
    if (tid == 0) first_bad = n;
    __syncthreads();
    for (int i = warp; i < n; i += PICK / 32) {
        const int row = s0 + i, x = a.drafts[row];
        const Row r = whole_row(a, heat, row);
        if (lane == 0) {
            bool fine = false;
            if (x < 0 || x >= a.V) atomicOr(a.err, ERR_TOKEN);
            else if (!r.none()) {
                if (greedy) fine = x == r.at;
                else {
                    const float z = a.x[row * a.ld + x];
                    double w = (double)heat(z, r.max), sum = r.sum;
                    if (a.cut && a.cut[row].on) sum = a.cut[row].total, w = z >= a.cut[row].least ? w : 0.0;
                    fine = (double)a.accept_u[row] * (a.q ? (double)a.q[row * a.ldq + x] : 1.0) < w / sum;
                }
            }
            if (!fine) atomicMin(&first_bad, i);
        }
    }
    __syncthreads();
    const int acc = first_bad, row = s0 + acc;
    if (warp == 0) {
        const Row r = whole_row(a, heat, row);
        if (lane == 0) row_sh = r;
    }
    if (rank == 0) {
        for (int i = tid; i <= n; i += PICK)
            if (i != acc) a.tokens[s0 + i] = i < acc ? a.drafts[s0 + i] : -1;
        if (tid == 0) a.accepted[e] = acc;
    }
    __syncthreads();
    const Row r = row_sh;
    if (r.none() || greedy) {
        if (rank == 0 && tid == 0) a.tokens[row] = r.none() ? -1 : r.at;
        return;
    }
    double sum = r.sum;
    float least = -INFINITY;
    if (a.cut && a.cut[row].on) sum = a.cut[row].total, least = a.cut[row].least;
    const double inv = 1.0 / sum;
    const float* x = a.x + row * a.ld;
    const float* q = a.q ? a.q + row * a.ldq : nullptr;
    const int drafted = a.drafts[row], shift = quad_shift(x);
    const bool aligned_q = q && (quad_shift(q) == shift);
    const int tiles_all = ((a.V + shift + 3) / 4 + PICK - 1) / PICK, per = (tiles_all + CLUSTER - 1) / CLUSTER;
    const int t0 = min(tiles_all, rank * per), t1 = min(tiles_all, t0 + per);
    bool rest = acc < n;
    // weights of the four logits of quad k of tile t
    auto weights = [&](int t, double (&w)[4]) {
        const int i = 4 * (t * PICK + tid) - shift;
        const float4 z4 = quad(x, i, a.V, -INFINITY);
        const float z[4] = {z4.x, z4.y, z4.z, z4.w};
        float4 q4 = make_float4(0.f, 0.f, 0.f, 0.f);
        if (rest && q) {
            if (aligned_q) q4 = quad(q, i, a.V, 0.f);
            else q4 = make_float4(i >= 0 && i < a.V ? q[i] : 0.f, i + 1 >= 0 && i + 1 < a.V ? q[i + 1] : 0.f, i + 2 >= 0 && i + 2 < a.V ? q[i + 2] : 0.f,
                                  i + 3 >= 0 && i + 3 < a.V ? q[i + 3] : 0.f);
        }
        const float qv[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            double p = z[j] >= least ? (double)heat(z[j], r.max) * inv : 0.0;
            if (rest) p -= q ? (double)qv[j] : (i + j == drafted ? 1.0 : 0.0);
            w[j] = p > 0.0 ? p : 0.0;
        }
    };
    double total;
    for (;;) {
        for (int t = t0; t < t1; ++t) {
            double w[4];
            weights(t, w);
            const double s = warp_sum((w[0] + w[1]) + (w[2] + w[3]));
            if (lane == 0) warp_part[warp] = s;
            __syncthreads();
            if (tid == 0) {
                double y = 0.0;
                for (int k = 0; k < PICK / 32; ++k) y += warp_part[k];
                tile_sum[t - t0] = y;
            }
            __syncthreads();
        }
        if (tid == 0) {
            double y = 0.0;
            for (int t = t0; t < t1; ++t) y += tile_sum[t - t0];
            cta_sum = y;
        }
        cl.sync();
        total = 0.0;
        for (int c = 0; c < CLUSTER; ++c) total += *cl.map_shared_rank(&cta_sum, c);
        if (!rest || total > 0.0) break;
        rest = false;                                       // nothing is left of the draft's excess: the target's own probabilities
        cl.sync();
    }
    const double target = (double)a.sample_u[e] * total;
    double before = 0.0, base = 0.0;
    int owner = -1;                                         // the CTA in whose share the sum passes the target (rounding: the last that has any)
    for (int c = 0; c < CLUSTER; ++c) {
        const double y = *cl.map_shared_rank(&cta_sum, c);
        if (y > 0.0) {
            owner = c, base = before;
            if (before + y > target) break;
        }
        before += y;
    }
    if (rank == owner) {
        int tile = t0;
        before = base;
        for (int t = t0; t < t1; ++t) {
            const double y = tile_sum[t - t0];
            if (y > 0.0) {
                tile = t, base = before;
                if (before + y > target) break;
            }
            before += y;
        }
        double w[4];
        weights(tile, w);
        double s = (w[0] + w[1]) + (w[2] + w[3]), own = s;
        const int i = 4 * (tile * PICK + tid) - shift;
        if (tid == 0) found = 0x7fffffff, last_some = -1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        if (lane == 31) warp_part[warp] = s;
        __syncthreads();
        for (int k = 0; k < warp; ++k) s += warp_part[k];
        scan[tid] = s;
        __syncthreads();
        double cum = base + (tid ? scan[tid - 1] : 0.0);
        if (own > 0.0) {
            int last = -1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                cum += w[j];
                if (w[j] > 0.0) {
                    last = i + j;
                    if (cum > target) {
                        atomicMin(&found, i + j);
                        break;
                    }
                }
            }
            atomicMax(&last_some, last);
        }
        __syncthreads();
        if (tid == 0) a.tokens[row] = found != 0x7fffffff ? found : last_some;
    }
    cl.sync();                                              // nobody's sums go while they are read
}

int slices_of(int R, int V, int& threads) {
    // Slices of 16384 logits where they fill the GPU twice, of 4096 otherwise
    threads = (int64_t)R * ((V + 3 + 16383) / 16384) >= 2 * 148 ? 1024 : 256;
    return (V + 3 + 16 * threads - 1) / (16 * threads);
}

}  // namespace

}  // namespace b200seq

using namespace b200seq;

extern "C" {

size_t b200seq_verify_scratch_bytes(int R, int V, int ruled) {
    if (R < 1 || V < 1 || V > MAX_V) return 0;
    int threads;
    return (size_t)R * slices_of(R, V, threads) * sizeof(Partial) + (ruled ? (size_t)R * sizeof(Cut) : 0);
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
    int threads;
    VerifyArgs a{logits, ld, R, V, B, 0, start, drafts, accept_u, sample_u, temperature, top_k, top_p, draft_probs, ldq, accepted, tokens, (Partial*)scratch, nullptr, error_flag_dev()};
    a.slices = slices_of(R, V, threads);
    if (ruled) a.cut = reinterpret_cast<Cut*>(a.part + (size_t)R * a.slices);
    const cudaStream_t cs = (cudaStream_t)stream;
    if (R > 0) {
        if (threads == 1024) launch_chained(row_stats_kernel<1024>, dim3(a.slices, R), 1024, 0, cs, a);
        else launch_chained(row_stats_kernel<256>, dim3(a.slices, R), 256, 0, cs, a);
        SEQ_LAUNCH_CHECK("verify_drafts");
        if (ruled) {
            launch_chained(row_cut_kernel, dim3(CLUSTER * R), CUT, 0, cs, a);
            SEQ_LAUNCH_CHECK("verify_drafts");
        }
    }
    launch_chained(pick_kernel, dim3(CLUSTER * B), PICK, 0, cs, a);
    SEQ_LAUNCH_CHECK("verify_drafts");
    return 0;
}

}  // extern "C"
