// seq_weigh_tc.cu -- the soft-max weight of cached keys from steps of many rows (a row: a token and a query head of the key head), on the 5th-generation tensor cores.
//
// Two launches of one kernel with its operands' places changed, so that what is reduced over is always a thread's own:
//   denominators (SUMS = false)  a CTA has 128 rows, walks over tiles of 64 keys; a thread has a row, its running maximum and sum of exponentials
//   sums (SUMS = true)           a CTA has 128 keys, walks over tiles of 64 rows; a thread has a key and adds 2^(score - the row's denominator) up, rows in their order
// No atomics, no scores in memory.  Scores are needed to 22 bits: every f32 operand is split into two f16 parts (x 2^4 = h + l), a product runs as l h', h l', h h'.  An
// operand is off by 2^-23 of itself or 2^-29, whichever is more; the queries carry the scale, so that a tile is scores in base 2.  Beyond 4094 an operand has no such parts:
// they make a row's or a key's sum NaN, and such a sum is made again by plain f32 products (plain_row, plain_key).
//
// Its floor is the tensor pipe, three products a pass: 6.3 MFLOP a tile of 128 x 64 at heads of 128, 0.55 us at the rate of an SM.  2047 tokens of 32 heads of 128 (8 key heads): 123 us,
// 15 of splitting and passes of 57 and 55, in which the pipe is active 54 and 57 % (31 a pass at its rate); where the rest of a pass goes has not been taken apart.  So that nothing else takes as long, rows and
// keys are split once, ahead of the two passes: tiles of 64 of them in the work area, two planes of f16 in the swizzled order of shared memory, so that a tile is one bulk copy.  (Split by
// loader warps each time a tile was needed: 4850 instructions of warps a tile, 90 us a pass of 2047 tokens.)  The operand that stays lies in TMEM (128 columns at most), the one that
// streams in three stages; 256 columns of TMEM and under 100 KB of shared memory: two CTAs an SM, so that one's beginning and end run beside the other's tiles.
//   warps 0 - 3   the resident operand to TMEM, then a thread a row of the accumulator     warp 4   copies     warp 5   issues the products
// Few row tiles or key tiles: the walk is cut into parts, whose (maximum, sum) are joined before the second pass, whose sums after it, in order.  Steps whose keys do not fit the work
// area go in several runs over entries and key heads.
// Every wait is bounded (tc_pair.cuh): one that runs out sets bit 1 of the error flags and the CTA leaves through the common exit.
#include "seq_weigh.cuh"
#include "tc_split.cuh"

namespace b200seq {

namespace {

using namespace tcsplit;

constexpr int NT = 64, MT = 128;                 // rows of the streamed tile, of the resident one
constexpr int PLANE = NT * 128;                  // bytes of one 64-row x 64-wide plane
constexpr int STAGES = 3;
constexpr int THREADS = 192;
constexpr int64_t KEYS_FLOATS = 64 << 20;        // of split keys in the work area, where a step has more of them than one entry's one head
constexpr float UP = 16.f, DOWN = 1.f / 256.f;   // operands times 2^4 each

struct TcArgs {
    WeighArgs w;
    int parts;                 // of this launch's walk
    int tiles;                 // denominators: row tiles of 128 (bound); sums: key tiles of 128
    int key_tiles;             // of 64, of the longest sequence
    int stage;                 // bytes of a split tile
    uint8_t *qtiles, *ktiles;  // split rows [entry][key head][tile]; split keys [entry - e0][key head - g0][tile]
    float* lse;                // [split rows]: base-2 logarithm of the denominator
    float2* stat;              // [part][split rows]: (maximum, sum) in base 2, where a walk has parts
    float* psum;               // sums, parts > 1: [part][entry - e0][key head - g0][key_room]
    int64_t qrows, key_room;   // split rows (bound); keys
    int e0, ne, g0, ng;        // the run's entries and key heads
};

// the tiles of `size` rows of entries e0 ..: which entry has tile idx, and its number there; by every warp for itself
__device__ __forceinline__ bool find_rows(const WeighArgs& a, const b200seq_step& st, int e0, int ne, int size, int idx, int& e, int& tile) {
    const int lane = threadIdx.x & 31, R = a.H / a.G;
    int acc = 0;
    for (int b0 = 0; b0 < ne; b0 += 32) {
        int n = 0;
        if (b0 + lane < ne) n = (WeighEntry(a, st, e0 + b0 + lane, false).n * R + size - 1) / size;
        int up = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += y;
        }
        const unsigned in = __ballot_sync(0xffffffffu, idx >= acc + up - n && idx < acc + up);
        if (in) {
            const int l = __ffs(in) - 1;
            e = e0 + b0 + l, tile = idx - acc - __shfl_sync(0xffffffffu, up - n, l);
            return true;
        }
        acc += __shfl_sync(0xffffffffu, up, 31);
    }
    return false;
}
// number of the first split tile of an entry's key head; by every warp for itself
__device__ __forceinline__ int first_qtile(const WeighArgs& a, const b200seq_step& st, int e, int n, int g) {
    const int lane = threadIdx.x & 31, R = a.H / a.G;
    int before = 0;
    for (int i = lane; i < e; i += 32) before += (WeighEntry(a, st, i, false).n * R + NT - 1) / NT;
    before = __reduce_add_sync(0xffffffffu, before);
    return before * a.G + g * ((n * R + NT - 1) / NT);
}

// whether the split tiles of an entry's key heads lie within the work area (not all do where the entries' tokens overlap: its size is that of tokens of one entry each); q0: of head g
__device__ __forceinline__ bool tiles_fit(const TcArgs& a, int q0, int g, int n, int R) { return q0 + (int64_t)(a.w.G - g) * ((n * R + NT - 1) / NT) <= a.qrows / NT; }

// the key tiles that a tile of rows (tokens at p_first .. p_last) sees, in their order
struct KeyWalk {
    int first, main0, total;
    __device__ __forceinline__ KeyWalk(const WeighArgs& a, int p_first, int p_last) {
        const WeighSpan s(a, p_first);
        first = min((s.keep + NT - 1) / NT, s.lo / NT);
        main0 = s.lo / NT;
        total = first + p_last / NT - main0 + 1;
    }
    __device__ __forceinline__ int key0(int tile) const { return (tile < first ? tile : main0 + tile - first) * NT; }
};
// rows (of `rows`) that see a key j: from .. to - 1
__device__ __forceinline__ void rows_of_key(const WeighArgs& a, const WeighEntry& en, int R, int rows, int j, int& from, int& to) {
    from = j > en.p0 ? (j - en.p0) * R : 0, to = rows;      // (products of at most the entry's rows: checked by the caller)
    if (a.window > 0 && j >= a.keep_first) to = (int)min((int64_t)rows, max((int64_t)0, ((int64_t)j + a.window - en.p0) * R));
    if (a.chunk > 0) to = (int)min((int64_t)to, max((int64_t)0, ((int64_t)(j / a.chunk + 1) * a.chunk - en.p0) * R));
    from = min(from, rows);
}

template <bool CAP>
__device__ __forceinline__ float score_of(const WeighArgs& a, float s) {
    return CAP ? a.softcap * WEIGH_LOG2E * tanhf(s * DOWN / a.softcap) : s * DOWN;
}

__device__ __forceinline__ void split16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h), lo = *reinterpret_cast<const uint32_t*>(&l);
}

// ---- plain forms, for sums that are no numbers ---------------------------------------------------------------------------------------------------
__device__ __noinline__ float2 plain_row(const WeighArgs& a, const b200seq_step& st, const WeighEntry& en, int e, int g, int row, const KeyWalk walk, int part, int parts, bool four) {
    const WeighSpan span(a, en.p0 + row / (a.H / a.G));
    float m = -INFINITY, l = 0.f;
    for (int t = part; t < walk.total; t += parts)
        for (int j = walk.key0(t); j < walk.key0(t) + NT; ++j) {
            if (!span.sees(j)) continue;
            const float z = plain_score(a, st, en, e, g, row, j, four);
            if (z > m) l = m == -INFINITY ? l : l * ex2(m - z), m = z;
            if (z != -INFINITY) l += ex2(z - m);
        }
    return make_float2(m, l);
}

// the base-2 logarithm of a sum; infinite where there is none: such a row gives nothing
__device__ __forceinline__ float lse_of(float m, float l) { return l != l ? l : m == -INFINITY ? INFINITY : m + log2f(l); }

// a thread a row: the parts of its walk (tiles that no entry has hold anything, and nobody reads theirs)
__global__ void __launch_bounds__(128) weigh_lse_kernel(const __grid_constant__ TcArgs a) {
    chain_enter();
    const int64_t row = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (row >= a.qrows) return;
    const float2* s = a.stat + row;
    float m = -INFINITY, l = 0.f;
#pragma unroll 8
    for (int i = 0; i < a.parts; ++i) m = fmaxf(m, s[i * a.qrows].x);
#pragma unroll 8
    for (int i = 0; i < a.parts; ++i) {
        const float2 x = s[i * a.qrows];
        l += x.x == -INFINITY ? x.y : x.y * ex2(x.x - m);
    }
    a.lse[row] = lse_of(m, l);
}

__device__ __noinline__ float plain_key(const TcArgs& a, const b200seq_step& st, const WeighEntry& en, int e, int g, int key, int tile0, int tiles, int part, int64_t qrow0, bool four) {
    const int R = a.w.H / a.w.G, rows = en.n * R;
    float sum = 0.f;
    for (int i = part; i < tiles; i += a.parts)
        for (int r = (tile0 + i) * NT; r < min(rows, (tile0 + i + 1) * NT); ++r) {
            const WeighSpan span(a.w, en.p0 + r / R);
            if (!span.sees(key)) continue;
            const float lse = a.lse[qrow0 + r];
            sum += ex2(plain_score(a.w, st, en, e, g, r, key, four) - lse);
        }
    return sum;
}

// Rows and keys split into tiles: grid (row tiles (bound) * key heads + key tiles * key heads * entries of the run); the former only in a step's first run
template <bool FOUR>
__global__ void __launch_bounds__(256) weigh_split_kernel(const __grid_constant__ TcArgs a, const __grid_constant__ b200seq_step st, int row_blocks) {
    chain_enter();
    __shared__ int64_t at_sh[NT];      // where a row's values lie; -1: there is none
    __shared__ float fac_sh[NT];
    __shared__ int par_sh[NT];
    const WeighArgs& w = a.w;
    const int tid = threadIdx.x, D = w.D, G = w.G, R = w.H / G, KB = (D + 63) >> 6, bs = st.block_size;
    const bool keys = (int)blockIdx.x >= row_blocks;
    uint8_t* out;
    if (!keys) {
        const int g = blockIdx.x % G;
        int e, tile;
        if (!find_rows(w, st, 0, st.B, NT, blockIdx.x / G, e, tile)) return;
        const WeighEntry en(w, st, e, false);
        const int q0 = first_qtile(w, st, e, en.n, g);
        if (!tiles_fit(a, q0, g, en.n, R)) return;
        out = a.qtiles + (int64_t)(q0 + tile) * a.stage;
        if (tid < NT) {
            const int row = tile * NT + tid;
            int64_t x = -1;
            if (row < en.n * R) {
                const int h = g * R + row % R;
                x = (int64_t)(en.t0 + row / R) * w.ld + (int64_t)h * D;
                fac_sh[tid] = weigh_factor(w, h) * (w.softcap > 0.f ? UP : UP * WEIGH_LOG2E);
            }
            at_sh[tid] = x;
        }
    } else {
        int i = blockIdx.x - row_blocks;
        const int tile = i % a.key_tiles;
        i /= a.key_tiles;
        const int g = a.g0 + i % a.ng, e = a.e0 + i / a.ng;
        const WeighEntry en(w, st, e, false);
        if (en.n == 0 || tile * NT >= en.keys) return;
        const WeighSpan span(w, en.p0);
        if ((tile + 1) * NT <= span.lo && tile * NT >= span.keep) return;      // (nobody sees them)
        out = a.ktiles + ((int64_t)i * a.key_tiles + tile) * a.stage;
        if (tid < NT) {
            const int key = tile * NT + tid;
            int64_t x = -1;
            if (key < en.keys) {
                const int page = kv4_page_read(st.block_table[(int64_t)e * st.max_blocks + key / bs], w.err), o = key % bs;
                if (FOUR) {
                    const Kv4Row k = kv4_row(page, o, bs, g, G, w.NG);
                    x = k.codes, par_sh[tid] = (int)(k.params - k.codes);
                } else {
                    x = (((int64_t)page * bs + o) * G + g) * D;
                }
            }
            at_sh[tid] = x, fac_sh[tid] = UP;
        }
    }
    __syncthreads();
    // 16 threads to a row's 64 values
    const int c4 = tid & 15, r0 = tid >> 4;
    for (int u = 0; u < KB; ++u) {
        const int d = u * 64 + c4 * 4;
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t at = at_sh[r0 + 16 * i];
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at < 0 || d >= D) continue;
            if (FOUR && keys) {
                const uint8_t* k = w.kpool4 + at;
                const uint32_t word = *reinterpret_cast<const uint32_t*>(k + 4 * ((d % 32 / 8) * w.NG + d / 32)) >> (4 * (d % 8));
                const uint32_t par = *reinterpret_cast<const uint32_t*>(k + par_sh[r0 + 16 * i] + 4 * (d / 32));
                const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&par));
                auto val = [&](uint32_t c) { return fmaf(__uint_as_float(c | 0x4B000000u) - 8388608.f, sm.x, sm.y); };
                x[i] = make_float4(val(word & 15u), val((word >> 4) & 15u), val((word >> 8) & 15u), val((word >> 12) & 15u));
            } else {
                x[i] = ld4((keys ? w.kpool : w.q) + at + d);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = r0 + 16 * i;
            const float f = at_sh[row] < 0 ? 0.f : fac_sh[row];
            uint32_t h0, h1, l0, l1;
            split16(x[i].x * f, x[i].y * f, h0, l0);
            split16(x[i].z * f, x[i].w * f, h1, l1);
            uint8_t* to = out + u * (2 * PLANE) + row * 128 + (((c4 >> 1) ^ (row & 7)) << 4) + ((c4 & 1) << 3);
            *reinterpret_cast<uint2*>(to) = make_uint2(h0, h1), *reinterpret_cast<uint2*>(to + PLANE) = make_uint2(l0, l1);
        }
    }
}

__device__ __forceinline__ void bulk_in(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// One pass.  Denominators: grid (row tiles * key heads, 1, parts); sums: grid (key tiles * parts * key heads * entries).
template <bool SUMS, bool CAP>
__global__ void __launch_bounds__(THREADS, 2) weigh_tc_kernel(const __grid_constant__ TcArgs a, const __grid_constant__ b200seq_step st, int four) {
    chain_enter();
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_base;
    __shared__ int abort_sh;
    __shared__ __align__(8) uint64_t bars[2 * STAGES + 5];
    __shared__ __align__(16) float lse_sh[STAGES][NT];
    const WeighArgs& w = a.w;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int R = w.H / w.G, KK = (w.D + 15) >> 4;
    const uint32_t ring = (sa(smem_raw) + 1023u) & ~1023u, stage = a.stage;
    const uint32_t B0 = sa(bars), b_full = B0, b_free = B0 + 8 * STAGES, acc_full = B0 + 16 * STAGES, acc_free = acc_full + 16, done = acc_free + 16;
    volatile int* ab = &abort_sh;
    // ---- what this CTA has ----
    int e, g, res0, part;                    // res0: first row or key of the resident operand
    if (!SUMS) {
        const int r = (int)blockIdx.x / a.ng;
        g = a.g0 + (int)blockIdx.x - r * a.ng, part = blockIdx.z;
        if (!find_rows(w, st, a.e0, a.ne, MT, a.tiles - 1 - r, e, res0)) return;      // (the last tiles see the most keys: first)
        res0 *= MT;
    } else {
        int i = blockIdx.x;
        const int eg = i % (a.ng * a.ne);
        i /= a.ng * a.ne;
        part = i % a.parts, res0 = i / a.parts * MT;                  // (the first keys are seen by the most rows)
        e = a.e0 + eg / a.ng, g = a.g0 + eg % a.ng;
    }
    const WeighEntry en(w, st, e, SUMS && res0 == 0 && part == 0 && g == 0 && threadIdx.x == 0);
    const int rows = en.n * R;
    if (en.n == 0 || (SUMS ? res0 >= en.keys : res0 >= rows)) return;
    const int q0 = first_qtile(w, st, e, en.n, g);
    if (!tiles_fit(a, q0, g, en.n, R)) return;
    const uint8_t *qt = a.qtiles + (int64_t)q0 * stage, *kt = a.ktiles + (int64_t)((e - a.e0) * a.ng + g - a.g0) * a.key_tiles * stage;
    const int last_row = min(rows, res0 + MT) - 1;
    const KeyWalk walk(w, SUMS ? 0 : en.p0 + res0 / R, SUMS ? 0 : en.p0 + last_row / R);
    int tile0 = 0, all = walk.total;         // sums: the row tiles from the first that sees one of the keys to the last
    if (SUMS) {
        int from, to, f2, t2;
        rows_of_key(w, en, R, rows, res0, from, to);
        rows_of_key(w, en, R, rows, min(res0 + MT, en.keys) - 1, f2, t2);
        to = w.window > 0 && res0 < w.keep_first ? rows : max(to, t2);
        tile0 = from / NT, all = to > from ? (to + NT - 1) / NT - tile0 : 0;
    }
    const int ntile = all > part ? (all - part + a.parts - 1) / a.parts : 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) bar_init(b_full + 8 * i, 1), bar_init(b_free + 8 * i, SUMS ? 5 : 1);
        for (int i = 0; i < 2; ++i) bar_init(acc_full + 8 * i, 1), bar_init(acc_free + 8 * i, 4);
        bar_init(done, 1);
        abort_sh = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(sa(&tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base, res = tmem + 2 * NT;               // columns: two accumulators | the resident operand's planes
    const uint32_t rplane = KK * 8;

    if (warp < 4) {
        // ===================== thread == row of the resident operand =====================
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const int mine = res0 + warp * 32 + lane, have = SUMS ? en.keys : rows;
        const bool live = mine < have;
        {   // its planes to TMEM (a tile of 64 that is not there: zeros)
            const bool there = (mine & ~(NT - 1)) < have;
            const int rr = mine & (NT - 1);
            const uint8_t* src = (SUMS ? kt : qt) + (int64_t)(mine / NT) * stage + rr * 128;
            for (int k0 = 0; k0 < KK; k0 += 4) {
                uint4 v[2][8];
#pragma unroll
                for (int c = 0; c < 8; ++c)
#pragma unroll
                    for (int p = 0; p < 2; ++p)
                        v[p][c] = there && k0 + (c >> 1) < KK ? *reinterpret_cast<const uint4*>(src + (k0 >> 2) * (2 * PLANE) + p * PLANE + ((c ^ (rr & 7)) << 4)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    if (k0 + kk >= KK) break;
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const uint4 x = v[p][2 * kk], y = v[p][2 * kk + 1];
                        const uint32_t r[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                        st8(res + lanes + p * rplane + (k0 + kk) * 8, r);
                    }
                }
            }
            st_wait();
            fence_before();
        }
        asm volatile("bar.sync 1, 160;" ::: "memory");                  // with the issuer
        float m = -INFINITY, l = 0.f;
        const WeighSpan span(w, SUMS ? 0 : en.p0 + (live ? mine : res0) / R);
        int from = 0, to = 0;
        if (SUMS) rows_of_key(w, en, R, rows, live ? mine : res0, from, to);
        bool ok = true;
        auto below = [](int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); };
#pragma unroll 1
        for (int j = 0; j < ntile; ++j) {
            const int t = part + j * a.parts, s = j % STAGES, n0 = SUMS ? (tile0 + t) * NT : walk.key0(t);
            // what of the tile this thread takes: [lo, hi), and those below kp
            const int lo = (SUMS ? from : span.lo) - n0, hi = (SUMS ? to : span.p + 1) - n0, kp = SUMS ? 0 : span.keep - n0;
            if (SUMS) ok = bar_wait<false>(b_full + 8 * s, (j / STAGES) & 1, ab);      // (its rows' denominators)
            ok = ok && bar_wait<false>(acc_full + 8 * (j & 1), (j >> 1) & 1, ab);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            float v[NT];
            ld32(tmem + lanes + (j & 1) * NT, v);
            ld32(tmem + lanes + (j & 1) * NT + 32, v + 32);
            ld_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(acc_free + 8 * (j & 1));
            if (CAP) {
#pragma unroll
                for (int i = 0; i < NT; ++i) v[i] = score_of<true>(w, v[i]);
            }
            if (!__all_sync(0xffffffffu, lo <= 0 && hi >= NT)) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t see = (below(hi - 32 * c) & ~below(lo - 32 * c)) | (below(hi - 32 * c) & below(kp - 32 * c));
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[32 * c + i] = (see >> i) & 1u ? v[32 * c + i] : -INFINITY;
                }
            }
            const uint64_t dn = CAP ? pk(1.f, 1.f) : pk(DOWN, DOWN);
            uint64_t sum[2] = {0, 0};
            if (!SUMS) {
                float m0 = fmaxf(v[0], v[1]), m1 = fmaxf(v[2], v[3]);
#pragma unroll
                for (int i = 4; i < NT; i += 4) m0 = fmaxf(m0, fmaxf(v[i], v[i + 1])), m1 = fmaxf(m1, fmaxf(v[i + 2], v[i + 3]));
                const float top = fmaxf(m, fmaxf(m0, m1) * (CAP ? 1.f : DOWN));
                const float off = top == -INFINITY ? 0.f : -top;
                l *= m == top ? 1.f : ex2(m - top);                     // (m = -inf: nothing yet, or a NaN that stays one)
                m = top;
                const uint64_t off2 = pk(off, off);
#pragma unroll
                for (int i = 0; i < NT; i += 2) {
                    float x, y;
                    upk(fma2(pk(v[i], v[i + 1]), dn, off2), x, y);
                    sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pk(ex2(x), ex2(y)));
                }
            } else {
#pragma unroll
                for (int i = 0; i < NT; i += 4) {
                    const float4 z = ld4(&lse_sh[s][i]);
                    float x, y;
                    upk(fma2(pk(v[i], v[i + 1]), dn, pk(-z.x, -z.y)), x, y);
                    sum[0] = add2(sum[0], pk(ex2(x), ex2(y)));
                    upk(fma2(pk(v[i + 2], v[i + 3]), dn, pk(-z.z, -z.w)), x, y);
                    sum[1] = add2(sum[1], pk(ex2(x), ex2(y)));
                }
                // The next copy into this place is of another proxy: these loads are before it only behind a fence.  (Without it a warp in 10^5 had a later tile's denominators.)
                async_fence();
                __syncwarp();
                if (lane == 0) bar_arrive(b_free + 8 * s);
            }
            float x, y;
            upk(add2(sum[0], sum[1]), x, y);
            l += x + y;
        }
        if (ok) {
            if (!SUMS) {
                if (mine < (rows + NT - 1) / NT * NT) {                 // (whole tiles: the places behind the last row give nothing)
                    float2 r = make_float2(m, l);
                    if (!live) r = make_float2(-INFINITY, 0.f);
                    else if (l != l) r = plain_row(w, st, en, e, g, mine, walk, part, a.parts, four);
                    if (live && w.sink && part == 0) {                  // the sink's term, once
                        const float sk = w.sink[g * R + mine % R] * WEIGH_LOG2E, top = fmaxf(r.x, sk);
                        if (top != -INFINITY) r = make_float2(top, (r.x == -INFINITY ? r.y : r.y * ex2(r.x - top)) + ex2(sk - top));      // (else neither has anything yet)
                    }
                    const int64_t row = (int64_t)q0 * NT + mine;
                    if (a.parts > 1) a.stat[part * a.qrows + row] = r;
                    else a.lse[row] = lse_of(r.x, r.y);
                }
            } else if (live) {
                if (l != l) l = plain_key(a, st, en, e, g, mine, tile0, all, part, (int64_t)q0 * NT, four);
                if (a.parts > 1) {
                    a.psum[((int64_t)(part * a.ne + e - a.e0) * a.ng + g - a.g0) * a.key_room + mine] = l;
                } else {
                    float* acc = w.acc + ((int64_t)en.slot * w.G + g) * w.acc_ld + mine;
                    *acc = mine < en.fresh ? *acc + l : l;
                }
            }
        }
    } else if (warp == 4) {
        // ===================== copies =====================
        if (elect()) {
            asm volatile("fence.proxy.async.global;" ::: "memory");     // (the tiles were written by ordinary stores)
            bool ok = true;
            int issued = 0;
#pragma unroll 1
            for (int j = 0; j < ntile && ok; ++j) {
                const int s = j % STAGES, t = part + j * a.parts;
                ok = bar_wait<false>(b_free + 8 * s, ((j / STAGES) & 1) ^ 1, ab);
                if (!ok) break;
                bar_expect(b_full + 8 * s, stage + (SUMS ? NT * 4 : 0));
                bulk_in(ring + s * stage, SUMS ? qt + (int64_t)(tile0 + t) * stage : kt + (int64_t)(walk.key0(t) / NT) * stage, stage, b_full + 8 * s);
                if (SUMS) bulk_in(sa(lse_sh[s]), a.lse + ((int64_t)q0 + tile0 + t) * NT, NT * 4, b_full + 8 * s);
                issued = j + 1;
            }
            // copies on their way land before the CTA goes (bounded)
            const unsigned long long t0 = now_ns();
            for (int j = max(0, issued - STAGES); j < issued; ++j)
                while (!bar_try<false>(b_full + 8 * (j % STAGES), (j / STAGES) & 1) && now_ns() - t0 < WAIT_NS) {}
        }
        __syncwarp();
    } else {
        // ===================== issuer =====================
        asm volatile("bar.sync 1, 160;" ::: "memory");
        if (elect()) {
            fence_after();
            constexpr uint32_t id = (1u << 4) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(MT >> 4) << 24);      // f16 operands, f32 sums
            bool ok = true;
#pragma unroll 1
            for (int j = 0; j < ntile && ok; ++j) {
                const int s = j % STAGES;
                ok = bar_wait<false>(b_full + 8 * s, (j / STAGES) & 1, ab) && (j < 2 || bar_wait<false>(acc_free + 8 * (j & 1), ((j - 2) >> 1) & 1, ab));
                if (!ok) break;
                fence_after();
                const uint64_t bd = desc_k128(ring + s * stage);
                const uint32_t d = tmem + (j & 1) * NT;
#pragma unroll
                for (int pr = 0; pr < 3; ++pr) {      // low x high, high x low, high x high
                    const uint32_t ra = res + (pr == 0 ? rplane : 0);
                    const int pb = pr == 1 ? PLANE : 0;
#pragma unroll 1
                    for (int kk = 0; kk < KK; ++kk)
                        mma_ts(d, ra + kk * 8, bd + (uint64_t)(((kk >> 2) * (2 * PLANE) + pb) / 16 + 2 * (kk & 3)), id, (pr | kk) != 0 ? 1u : 0u);
                }
                commit_one(acc_full + 8 * (j & 1));
                commit_one(b_free + 8 * s);
            }
            if (!ok) {      // what was issued reads shared memory and TMEM: wait for it (bounded) before the CTA goes
                commit_one(done);
                const unsigned long long t0 = now_ns();
                while (!bar_try<false>(done, 0) && now_ns() - t0 < WAIT_NS) {}
            }
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && abort_sh) atomicOr(w.err, 2);
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
    }
}

// the parts' sums, in their order; grid (blocks of 256 keys, key heads, entries of the run)
__global__ void __launch_bounds__(256) weigh_parts_kernel(const __grid_constant__ TcArgs a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    const int e = a.e0 + blockIdx.z, g = a.g0 + blockIdx.y, key = blockIdx.x * 256 + threadIdx.x;
    const WeighEntry en(a.w, st, e, false);
    if (en.n == 0 || key >= en.keys) return;
    float s = 0.f;
    for (int p = 0; p < a.parts; ++p) s += a.psum[((int64_t)(p * a.ne + blockIdx.z) * a.ng + blockIdx.y) * a.key_room + key];
    float* acc = a.w.acc + ((int64_t)en.slot * a.w.G + g) * a.w.acc_ld + key;
    *acc = key < en.fresh ? *acc + s : s;
}

template <bool SUMS, bool CAP>
cudaError_t run_one(const TcArgs& a, const b200seq_step& st, dim3 grid, bool four, cudaStream_t cs) {
    const int smem = STAGES * a.stage + 1024;
    cudaError_t e = cudaFuncSetAttribute(weigh_tc_kernel<SUMS, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    launch_chained(weigh_tc_kernel<SUMS, CAP>, grid, THREADS, smem, cs, a, st, (int)four);
    return cudaGetLastError();
}
template <bool SUMS>
cudaError_t run(const TcArgs& a, const b200seq_step& st, dim3 grid, bool four, cudaStream_t cs) {
    return a.w.softcap > 0.f ? run_one<SUMS, true>(a, st, grid, four, cs) : run_one<SUMS, false>(a, st, grid, four, cs);
}

}  // namespace

WeighTcPlan weigh_tc_plan(const b200seq_step& st, int H, int G, int D, int last, int64_t keys) {
    WeighTcPlan p;
    const int sms = 148, R = H / G;
    const int64_t each = (st.T + st.B - 1) / st.B, tokens = last > 0 && last < each ? last : each, rows = tokens * R;      // (were all entries equally long)
    const int64_t all = last > 0 ? (int64_t)last * st.B < st.T ? (int64_t)last * st.B : st.T : st.T;
    p.tiles = (int)((all * R + MT - 1) / MT + st.B - 1);
    p.qtiles = (int)((all * R + NT - 1) / NT + st.B - 1);
    p.stage = (D + 63) / 64 * 2 * PLANE;
    p.key_tiles = (int)((keys + NT - 1) / NT);
    p.key_room = (int64_t)(p.key_tiles + 1) / 2 * MT;
    // runs: as many entries, then as many key heads, as the work area has room for
    const int64_t tile = p.stage / 4;
    p.ne = st.B, p.ng = G;
    while (p.key_tiles * tile * p.ne * p.ng > KEYS_FLOATS && p.ne > 1) p.ne = (p.ne + 1) / 2;
    while (p.key_tiles * tile * p.ne * p.ng > KEYS_FLOATS && p.ng > 1) p.ng = (p.ng + 1) / 2;
    // Denominators: two CTAs an SM; a walk is cut where there are fewer, into parts of four key tiles at least.
    const int64_t units = (int64_t)p.ne * p.ng * ((rows + MT - 1) / MT);
    auto clamp = [](int64_t x, int64_t most) { return (int)(x < 1 || most < 1 ? 1 : x < most ? x : most); };
    const int64_t by_keys = p.key_tiles / 4;
    p.stat_parts = clamp(2 * sms / units, by_keys < 32 ? by_keys : 32);
    // Sums: the keys seen by most rows take twice the average, so that twice as many CTAs as fit are asked for; parts of eight row tiles at least.
    const int64_t row_tiles = (rows + NT - 1) / NT, by_rows = row_tiles / 8, cells = (int64_t)p.ne * p.ng * (p.key_room / MT);
    p.parts = clamp(4 * sms / cells, by_rows < 8 ? by_rows : 8);
    p.q_floats = (int64_t)p.qtiles * G * tile, p.k_floats = (int64_t)p.key_tiles * p.ne * p.ng * tile;
    p.lse_floats = (int64_t)p.qtiles * G * NT;
    p.stat_floats = p.stat_parts > 1 ? 2 * p.lse_floats * p.stat_parts : 0;
    p.floats = (size_t)(p.q_floats + p.k_floats + p.lse_floats + p.stat_floats + (p.parts > 1 ? p.parts * p.ne * p.ng * p.key_room : 0));
    return p;
}

bool weigh_tc_takes(const WeighArgs& w, bool four) {
    auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    return w.D <= 128 && w.D % 4 == 0 && w.ld % 4 == 0 && al(w.q) && (four || al(w.kpool));
}

int weigh_tc(const WeighArgs& w, const b200seq_step& st, const WeighTcPlan& p, float* scratch, bool four, cudaStream_t cs) {
    TcArgs a = {};
    a.w = w, a.key_tiles = p.key_tiles, a.stage = p.stage, a.key_room = p.key_room, a.qrows = p.lse_floats;
    a.qtiles = reinterpret_cast<uint8_t*>(scratch), a.ktiles = reinterpret_cast<uint8_t*>(scratch + p.q_floats);
    a.lse = scratch + p.q_floats + p.k_floats, a.stat = reinterpret_cast<float2*>(a.lse + p.lse_floats), a.psum = a.lse + p.lse_floats + p.stat_floats;
    for (int e0 = 0; e0 < st.B; e0 += p.ne)
        for (int g0 = 0; g0 < w.G; g0 += p.ng) {
            a.e0 = e0, a.ne = st.B - e0 < p.ne ? st.B - e0 : p.ne, a.g0 = g0, a.ng = w.G - g0 < p.ng ? w.G - g0 : p.ng;
            const int64_t row_blocks = e0 == 0 && g0 == 0 ? (int64_t)p.qtiles * w.G : 0, blocks = row_blocks + (int64_t)p.key_tiles * a.ng * a.ne;
            const int64_t b0 = (int64_t)p.tiles * a.ng, b1 = p.key_room / MT * p.parts * a.ng * a.ne;
            if (blocks > 0x7fffffff || b0 > 0x7fffffff || b1 > 0x7fffffff) return fail(B200SEQ_ERR_UNSUPPORTED, "key_weights: too many tiles for one launch");
            if (four) launch_chained(weigh_split_kernel<true>, dim3((unsigned)blocks), 256, 0, cs, a, st, (int)row_blocks);
            else launch_chained(weigh_split_kernel<false>, dim3((unsigned)blocks), 256, 0, cs, a, st, (int)row_blocks);
            SEQ_LAUNCH_CHECK("key_weights");
            a.parts = p.stat_parts, a.tiles = p.tiles;
            cudaError_t e = run<false>(a, st, dim3((unsigned)b0, 1, p.stat_parts), four, cs);
            if (e != cudaSuccess) return cuda_status(e, "key_weights");
            count_launch();
            if (p.stat_parts > 1) {
                launch_chained(weigh_lse_kernel, dim3((unsigned)((a.qrows + 127) / 128)), 128, 0, cs, a);
                SEQ_LAUNCH_CHECK("key_weights");
            }
            a.parts = p.parts, a.tiles = (int)(p.key_room / MT);
            e = run<true>(a, st, dim3((unsigned)b1), four, cs);
            if (e != cudaSuccess) return cuda_status(e, "key_weights");
            count_launch();
            if (p.parts > 1) {
                launch_chained(weigh_parts_kernel, dim3((unsigned)((p.key_room + 255) / 256), a.ng, a.ne), 256, 0, cs, a, st);
                SEQ_LAUNCH_CHECK("key_weights");
            }
        }
    return 0;
}

}  // namespace b200seq
