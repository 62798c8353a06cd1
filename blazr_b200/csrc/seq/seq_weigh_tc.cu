// seq_weigh_tc.cu -- the soft-max weight of cached keys from steps of many rows (a row: a token and a query head of the key head), on the 5th-generation tensor cores.
//
// Two launches of one kernel with its operands' places changed, so that what is reduced over is always a thread's own:
//   denominators (SUMS = false)  a CTA has 128 rows, walks over tiles of 64 keys; a thread has a row, its running maximum and sum of exponentials
//   sums (SUMS = true)           a CTA has 128 keys, walks over tiles of 64 rows; a thread has a key and adds 2^(score - the row's denominator) up, rows in their order
// No atomics, no scores in memory.  Scores are needed to 22 bits: every f32 operand is split into two f16 parts (x 2^4 = h + l), a product runs as l h', h l', h h'.  An
// operand is off by 2^-23 of itself or 2^-29, whichever is more; the queries carry the scale, so that a tile is scores in base 2.  Beyond 4094 an operand has no such parts:
// they make a row's or a key's sum NaN, and such a sum is made again by plain f32 products (plain_row, plain_key).
//
// What bounds it is the tensor pipe, three products a pass: 6.3 MFLOP a tile of 128 x 64 at heads of 128, 0.55 us at the rate of an SM.  The operand that stays lies in TMEM
// (128 columns at most), the one that streams goes through shared memory, fetched, split and swizzled by four warps (rows lie anywhere: pages, heads).  256 columns of TMEM and
// under 100 KB of shared memory: two CTAs an SM, so that one's beginning and end run beside the other's tiles.
//   warps 0 - 3   the resident operand to TMEM, then a thread a row of the accumulator     warps 4 - 7   loaders     warp 8   issues the products
// Few row tiles or key tiles: the walk is cut into parts, whose (maximum, sum) the second launch joins, whose sums a third one adds up in order.
// Every wait is bounded (tc_pair.cuh): one that runs out sets bit 1 of the error flags and the CTA leaves through the common exit.
#include "seq_weigh.cuh"
#include "tc_split.cuh"

namespace b200seq {

namespace {

using namespace tcsplit;

constexpr int NT = 64, MT = 128;                 // rows of the streamed tile, of the resident one
constexpr int PLANE = NT * 128;                  // bytes of one 64-row x 64-wide plane
constexpr int STAGES = 3;
constexpr int THREADS = 288;
constexpr float UP = 16.f, DOWN = 1.f / 256.f;   // operands times 2^4 each

struct TcArgs {
    WeighArgs w;
    int parts, stat_parts;     // of this launch's walk; of the denominators' walk
    int tiles;                 // denominators: row tiles (bound); sums: key tiles
    float2* stat;              // [T * H][stat_parts]: (maximum, sum) in base 2, where a walk has parts
    float* psum;               // sums, parts > 1: [part][B][G][key_room]
    int64_t key_room;
    int B;
};

// which of the entries' row tiles: its entry and first row; by every warp for itself
__device__ __forceinline__ bool find_rows(const WeighArgs& a, const b200seq_step& st, int idx, int& e, int& row0) {
    const int lane = threadIdx.x & 31, R = a.H / a.G;
    int acc = 0;
    for (int b0 = 0; b0 < st.B; b0 += 32) {
        int n = 0;
        if (b0 + lane < st.B) n = (WeighEntry(a, st, b0 + lane, false).n * R + MT - 1) / MT;
        int up = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += y;
        }
        const unsigned in = __ballot_sync(0xffffffffu, idx >= acc + up - n && idx < acc + up);
        if (in) {
            const int l = __ffs(in) - 1;
            e = b0 + l, row0 = (idx - acc - __shfl_sync(0xffffffffu, up - n, l)) * MT;
            return true;
        }
        acc += __shfl_sync(0xffffffffu, up, 31);
    }
    return false;
}

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

// a row's denominator (base-2 logarithm) from its maximum and sum; infinite where the row gives nothing
__device__ __forceinline__ float lse_of(const WeighArgs& w, int h, float m, float l) {
    if (l != l) return l;
    const float v = weigh_lse(w, h, m, l);
    return v == -INFINITY ? INFINITY : v;
}
// a thread a row: the parts of its walk (rows that do not count have none, and nobody reads theirs)
__global__ void __launch_bounds__(128) weigh_lse_kernel(const __grid_constant__ TcArgs a, int rows) {
    chain_enter();
    const int row = blockIdx.x * 128 + threadIdx.x;
    if (row >= rows) return;
    const float2* s = a.stat + (int64_t)row * a.stat_parts;
    float m = -INFINITY, l = 0.f;
#pragma unroll 8
    for (int i = 0; i < a.stat_parts; ++i) m = fmaxf(m, s[i].x);
#pragma unroll 8
    for (int i = 0; i < a.stat_parts; ++i) {
        const float2 x = s[i];
        l += x.x == -INFINITY ? x.y : x.y * ex2(x.x - m);
    }
    a.w.lse[row] = lse_of(a.w, row % a.w.H, m, l);
}

__device__ __noinline__ float plain_key(const TcArgs& a, const b200seq_step& st, const WeighEntry& en, int e, int g, int key, int tile0, int tiles, int part, bool four) {
    const int R = a.w.H / a.w.G, rows = en.n * R;
    float sum = 0.f;
    for (int i = part; i < tiles; i += a.parts)
        for (int r = (tile0 + i) * NT; r < min(rows, (tile0 + i + 1) * NT); ++r) {
            const WeighSpan span(a.w, en.p0 + r / R);
            if (!span.sees(key)) continue;
            const float lse = a.w.lse[(int64_t)(en.t0 + r / R) * a.w.H + g * R + r % R];
            sum += ex2(plain_score(a.w, st, en, e, g, r, key, four) - lse);
        }
    return sum;
}

// One launch.  Denominators: grid (row tiles * key heads, 1, parts); sums: grid (key tiles * parts * key heads * entries).
template <bool SUMS, bool FOUR, bool CAP>
__global__ void __launch_bounds__(THREADS, 2) weigh_tc_kernel(const __grid_constant__ TcArgs a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_base;
    __shared__ int abort_sh;
    __shared__ __align__(8) uint64_t bars[2 * STAGES + 5];
    __shared__ __align__(16) float lse_sh[STAGES][NT];
    __shared__ int64_t row_sh[3][NT];                                   // loaders: where the rows of three tiles lie,
    __shared__ float fac_sh[SUMS ? 3 : 1][NT];                          // their factors,
    __shared__ int par_sh[FOUR ? 3 : 1][NT];                            // their parameters behind their codes
    const WeighArgs& w = a.w;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int D = w.D, G = w.G, R = w.H / w.G, KB = (D + 63) >> 6, KK = (D + 15) >> 4;
    const uint32_t ring = (sa(smem_raw) + 1023u) & ~1023u, stage = KB * 2 * PLANE;
    const uint32_t B0 = sa(bars), b_full = B0, b_free = B0 + 8 * STAGES, acc_full = B0 + 16 * STAGES, acc_free = acc_full + 16, done = acc_free + 16;
    volatile int* ab = &abort_sh;
    // ---- what this CTA has ----
    int e, g, res0, part;                    // res0: first row or key of the resident operand
    if (!SUMS) {
        const int r = (int)blockIdx.x / G;
        g = (int)blockIdx.x - r * G, part = blockIdx.z;
        if (!find_rows(w, st, a.tiles - 1 - r, e, res0)) return;      // (the last tiles see the most keys: first)
    } else {
        int i = blockIdx.x;
        const int eg = i % (G * a.B);
        i /= G * a.B;
        part = i % a.parts, res0 = i / a.parts * MT;                  // (the first keys are seen by the most rows)
        e = eg / G, g = eg - e * G;
    }
    const WeighEntry en(w, st, e, SUMS && res0 == 0 && part == 0 && g == 0 && threadIdx.x == 0);
    const int rows = en.n * R;
    if (en.n == 0 || (SUMS ? res0 >= en.keys : res0 >= rows)) return;
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
    const int32_t* bt = st.block_table + (int64_t)e * st.max_blocks;
    const int bs = st.block_size;
    const float fold = CAP ? UP : UP * WEIGH_LOG2E;      // a query's factor beside its head's scale
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) bar_init(b_full + 8 * i, 4), bar_init(b_free + 8 * i, SUMS ? 5 : 1);
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
        const int mine = res0 + warp * 32 + lane;
        const bool live = SUMS ? mine < en.keys : mine < rows;
        {
            const int at = live ? mine : res0;
            const float* src = nullptr;
            Kv4Row k4{0, 0};
            float f = UP;
            if (SUMS) {
                const int page = kv4_page_read(bt[at / bs], w.err), o = at % bs;
                if (FOUR) k4 = kv4_row(page, o, bs, g, G, w.NG);
                else src = w.kpool + (((int64_t)page * bs + o) * G + g) * D;
            } else {
                const int h = g * R + at % R;
                src = w.q + (int64_t)(en.t0 + at / R) * w.ld + (int64_t)h * D;
                f = weigh_factor(w, h) * fold;
            }
            if (!live) f = 0.f;
            if (SUMS && FOUR) {
#pragma unroll 2
                for (int kk = 0; kk < KK; ++kk) {
                    const int grp = kk >> 1;
                    const uint32_t par = *reinterpret_cast<const uint32_t*>(w.kpool4 + k4.params + 4 * grp);
                    const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&par));
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t word = *reinterpret_cast<const uint32_t*>(w.kpool4 + k4.codes + 4 * ((2 * (kk & 1) + c) * w.NG + grp));
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = live && 16 * kk + 8 * c + i < D ? fmaf((float)((word >> (4 * i)) & 15u), sm.x, sm.y) * f : 0.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) split16(x[2 * i], x[2 * i + 1], hi[4 * c + i], lo[4 * c + i]);
                    }
                    st8(res + lanes + kk * 8, hi), st8(res + lanes + rplane + kk * 8, lo);
                }
            } else {
                for (int k0 = 0; k0 < KK; k0 += 4) {       // (the loads of 64 values at once: a chain of them is what a short walk would wait for)
                    float4 v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = live && 16 * k0 + 4 * i < D ? ld4(src + 16 * k0 + 4 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        if (k0 + kk >= KK) break;
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float4 x = v[4 * kk + i];
                            split16(x.x * f, x.y * f, hi[2 * i], lo[2 * i]), split16(x.z * f, x.w * f, hi[2 * i + 1], lo[2 * i + 1]);
                        }
                        st8(res + lanes + (k0 + kk) * 8, hi), st8(res + lanes + rplane + (k0 + kk) * 8, lo);
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
        for (int j = 0; j < ntile && ok; ++j) {
            const int t = part + j * a.parts, s = j % STAGES, n0 = SUMS ? (tile0 + t) * NT : walk.key0(t);
            // what of the tile this thread takes: [lo, hi), and those below kp
            const int lo = (SUMS ? from : span.lo) - n0, hi = (SUMS ? to : span.p + 1) - n0, kp = SUMS ? 0 : span.keep - n0;
            if (SUMS) ok = bar_wait<false>(b_full + 8 * s, (j / STAGES) & 1, ab);      // (its rows' denominators)
            ok = ok && bar_wait<false>(acc_full + 8 * (j & 1), (j >> 1) & 1, ab);
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float v[32];
                ld32(tmem + lanes + (j & 1) * NT + 32 * c, v);
                ld_wait();
                if (CAP) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = score_of<true>(w, v[i]);
                }
                const bool whole = __all_sync(0xffffffffu, lo <= 32 * c && hi >= 32 * c + 32);
                if (!whole) {
                    const uint32_t see = (below(hi - 32 * c) & ~below(lo - 32 * c)) | (below(hi - 32 * c) & below(kp - 32 * c));
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = (see >> i) & 1u ? v[i] : -INFINITY;
                }
                const uint64_t dn = CAP ? pk(1.f, 1.f) : pk(DOWN, DOWN);
                uint64_t sum = 0;
                if (!SUMS) {
                    float m0 = fmaxf(v[0], v[1]), m1 = fmaxf(v[2], v[3]);
#pragma unroll
                    for (int i = 4; i < 32; i += 4) m0 = fmaxf(m0, fmaxf(v[i], v[i + 1])), m1 = fmaxf(m1, fmaxf(v[i + 2], v[i + 3]));
                    const float top = fmaxf(m, fmaxf(m0, m1) * (CAP ? 1.f : DOWN));
                    const float off = top == -INFINITY ? 0.f : -top;
                    l *= m == top ? 1.f : ex2(m - top);                 // (m = -inf: nothing yet, or a NaN that stays one)
                    m = top;
                    const uint64_t off2 = pk(off, off);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float x, y;
                        upk(fma2(pk(v[i], v[i + 1]), dn, off2), x, y);
                        sum = add2(sum, pk(ex2(x), ex2(y)));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 z = ld4(&lse_sh[s][32 * c + i]);
                        float x, y;
                        upk(fma2(pk(v[i], v[i + 1]), dn, pk(-z.x, -z.y)), x, y);
                        sum = add2(sum, pk(ex2(x), ex2(y)));
                        upk(fma2(pk(v[i + 2], v[i + 3]), dn, pk(-z.z, -z.w)), x, y);
                        sum = add2(sum, pk(ex2(x), ex2(y)));
                    }
                }
                float x, y;
                upk(sum, x, y);
                l += x + y;
            }
            fence_before();
            __syncwarp();
            if (lane == 0) {
                bar_arrive(acc_free + 8 * (j & 1));
                if (SUMS) bar_arrive(b_free + 8 * s);
            }
        }
        if (ok && live) {
            if (!SUMS) {
                float2 r = make_float2(m, l);
                if (l != l) r = plain_row(w, st, en, e, g, mine, walk, part, a.parts, FOUR);
                const int h = g * R + mine % R;
                const int64_t row = (int64_t)(en.t0 + mine / R) * w.H + h;
                if (a.parts > 1) a.stat[row * a.parts + part] = r;
                else w.lse[row] = lse_of(w, h, r.x, r.y);
            } else {
                if (l != l) l = plain_key(a, st, en, e, g, mine, tile0, all, part, FOUR);
                if (a.parts > 1) {
                    a.psum[(((int64_t)part * a.B + e) * G + g) * a.key_room + mine] = l;
                } else {
                    float* acc = w.acc + ((int64_t)en.slot * G + g) * w.acc_ld + mine;
                    *acc = mine < en.fresh ? *acc + l : l;
                }
            }
        }
    } else if (warp < 8) {
        // ===================== loaders: 128 threads =====================
        // A unit is a 64-wide block of a tile: eight 16-byte pieces a thread, 16 lanes to a row's 64 values.  The next unit's loads are in flight while this one is split and
        // stored.  Where a tile's rows lie stands in a table in shared memory that 64 threads write a tile ahead, from pages asked for a tile before that.  (Looked up by every lane and
        // handed round by shuffles it was what the kernel spent its time on.)
        const int lw = warp - 4, lt = threadIdx.x - 128, hw = lw * 2 + (lane >> 4), c4 = lane & 15;
        auto row_of = [&](int j) { return (SUMS ? (tile0 + part + j * a.parts) * NT : walk.key0(part + j * a.parts)) + lt; };
        auto page_of = [&](int j) {      // (keys: the page of row lt of tile j)
            const int n = row_of(j);
            return !SUMS && n < en.keys ? kv4_page_read(bt[n / bs], w.err) : 0;
        };
        auto note = [&](int j, int page) {
            const int n = row_of(j), at = j % 3;
            int64_t x = -1;
            if (SUMS) {
                if (n < rows) {
                    const int h = g * R + n % R;
                    x = (int64_t)(en.t0 + n / R) * w.ld + (int64_t)h * D;
                    fac_sh[at][lt] = weigh_factor(w, h) * fold;
                }
            } else if (n < en.keys) {
                const int o = n % bs;
                if (FOUR) {
                    const Kv4Row k = kv4_row(page, o, bs, g, G, w.NG);
                    x = k.codes, par_sh[at][lt] = (int)(k.params - k.codes);
                } else {
                    x = (((int64_t)page * bs + o) * G + g) * D;
                }
            }
            row_sh[at][lt] = x;
        };
        auto fetch = [&](int j, int u, float4 (&x)[8]) {
            const int d = u * 64 + c4 * 4, at = j % 3;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t r = row_sh[at][hw + 8 * i];
                x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < 0 || d >= D) continue;
                if (!SUMS && FOUR) {
                    const uint8_t* k = w.kpool4 + r;
                    const uint32_t word = *reinterpret_cast<const uint32_t*>(k + 4 * ((d % 32 / 8) * w.NG + d / 32)) >> (4 * (d % 8));
                    const uint32_t par = *reinterpret_cast<const uint32_t*>(k + par_sh[at][hw + 8 * i] + 4 * (d / 32));
                    // (kept as they are until the values are needed; a word of a row that is one is told apart by bit 16)
                    x[i].x = __uint_as_float((word & 0xFFFFu) | 0x10000u), x[i].y = __uint_as_float(par);
                } else {
                    x[i] = ld4((SUMS ? w.q : w.kpool) + r + d);
                }
            }
        };
        int page = 0;
        float4 cur[8], nxt[8];
        if (lt < 64 && ntile > 0) note(0, page_of(0));
        if (lt < 64 && ntile > 1) page = page_of(1);
        asm volatile("bar.sync 2, 128;" ::: "memory");
        if (ntile > 0) fetch(0, 0, nxt);
        bool ok = true;
#pragma unroll 1
        for (int j = 0; j < ntile; ++j) {      // (a wait that ran out: the warps meet at their barrier all the same, to the end)
            const int s = j % STAGES;
            const bool more = j + 1 < ntile;
            float lse = INFINITY;
            if (lt < 64) {
                if (more) note(j + 1, page);
                if (j + 2 < ntile) page = page_of(j + 2);
                if (SUMS) {
                    const int n = row_of(j);
                    if (n < rows) lse = w.lse[(int64_t)(en.t0 + n / R) * w.H + g * R + n % R];
                }
            }
            asm volatile("bar.sync 2, 128;" ::: "memory");      // (three tables: nobody reads the one that is written next but one)
            if (!ok) continue;
#pragma unroll 1
            for (int u = 0; u < KB; ++u) {
#pragma unroll
                for (int i = 0; i < 8; ++i) cur[i] = nxt[i];
                const bool here = u + 1 < KB;
                if (here || more) fetch(here ? j : j + 1, here ? u + 1 : 0, nxt);
                if (u == 0) {
                    ok = bar_wait<false>(b_free + 8 * s, ((j / STAGES) & 1) ^ 1, ab);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (SUMS && lt < 64) lse_sh[s][lt] = lse;
                }
                uint32_t at = ring + s * stage + u * (2 * PLANE) + hw * 128 + (((c4 >> 1) ^ (hw & 7)) << 4) + ((c4 & 1) << 3);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float4 x = cur[i];
                    if (!SUMS && FOUR) {
                        const uint32_t word = __float_as_uint(x.x), par = __float_as_uint(x.y);
                        const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&par));
                        auto val = [&](uint32_t c) { return fmaf(__uint_as_float(c | 0x4B000000u) - 8388608.f, sm.x, sm.y); };
                        x = word & 0x10000u ? make_float4(val(word & 15u), val((word >> 4) & 15u), val((word >> 8) & 15u), val((word >> 12) & 15u)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    const float f = SUMS ? fac_sh[j % 3][hw + 8 * i] : UP;
                    const uint64_t f2 = pk(f, f);
                    float a0, a1, a2, a3;
                    upk(mul2(pk(x.x, x.y), f2), a0, a1), upk(mul2(pk(x.z, x.w), f2), a2, a3);
                    uint32_t h0, h1, l0, l1;
                    split16(a0, a1, h0, l0);
                    split16(a2, a3, h1, l1);
                    sts8(at, h0, h1), sts8(at + PLANE, l0, l1);
                    at += 8 * 128;
                }
            }
            if (!ok) continue;
            async_fence();
            __syncwarp();
            if (lane == 0) bar_arrive(b_full + 8 * s);
        }
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

// the parts' sums, in their order; grid (blocks of 256 keys, key heads, entries)
__global__ void __launch_bounds__(256) weigh_parts_kernel(const __grid_constant__ TcArgs a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    const int e = blockIdx.z, g = blockIdx.y, key = blockIdx.x * 256 + threadIdx.x;
    const WeighEntry en(a.w, st, e, false);
    if (en.n == 0 || key >= en.keys) return;
    float s = 0.f;
    for (int p = 0; p < a.parts; ++p) s += a.psum[(((int64_t)p * a.B + e) * a.w.G + g) * a.key_room + key];
    float* acc = a.w.acc + ((int64_t)en.slot * a.w.G + g) * a.w.acc_ld + key;
    *acc = key < en.fresh ? *acc + s : s;
}

template <bool SUMS, bool FOUR, bool CAP>
cudaError_t run_one(const TcArgs& a, const b200seq_step& st, dim3 grid, cudaStream_t cs) {
    const int smem = STAGES * ((a.w.D + 63) / 64) * 2 * PLANE + 1024;
    cudaError_t e = cudaFuncSetAttribute(weigh_tc_kernel<SUMS, FOUR, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    launch_chained(weigh_tc_kernel<SUMS, FOUR, CAP>, grid, THREADS, smem, cs, a, st);
    return cudaGetLastError();
}
template <bool SUMS>
cudaError_t run(const TcArgs& a, const b200seq_step& st, dim3 grid, bool four, cudaStream_t cs) {
    const bool cap = a.w.softcap > 0.f;
    if (four) return cap ? run_one<SUMS, true, true>(a, st, grid, cs) : run_one<SUMS, true, false>(a, st, grid, cs);
    return cap ? run_one<SUMS, false, true>(a, st, grid, cs) : run_one<SUMS, false, false>(a, st, grid, cs);
}

}  // namespace

WeighTcPlan weigh_tc_plan(const b200seq_step& st, int H, int G, int last, int64_t keys) {
    WeighTcPlan p;
    const int sms = 148, R = H / G;
    const int64_t each = (st.T + st.B - 1) / st.B, tokens = last > 0 && last < each ? last : each, rows = tokens * R;      // (were all entries equally long)
    const int64_t all = last > 0 ? (int64_t)last * st.B < st.T ? (int64_t)last * st.B : st.T : st.T;
    p.tiles = (int)((all * R + MT - 1) / MT + st.B - 1);
    // Denominators: two CTAs an SM; a walk is cut where there are fewer, into parts of four key tiles at least.
    const int64_t units = (int64_t)st.B * G * ((rows + MT - 1) / MT);
    auto clamp = [](int64_t x, int64_t most) { return (int)(x < 1 || most < 1 ? 1 : x < most ? x : most); };
    const int64_t key_tiles = (keys + NT - 1) / NT, by_keys = key_tiles / 4;
    p.stat_parts = clamp(2 * sms / units, by_keys < 32 ? by_keys : 32);
    // Sums: the keys seen by most rows take twice the average, so that twice as many CTAs as fit are asked for; parts of eight row tiles at least.
    p.key_tiles = (int)((keys + MT - 1) / MT);
    const int64_t row_tiles = (rows + NT - 1) / NT, by_rows = row_tiles / 8, cells = (int64_t)st.B * G * p.key_tiles;
    p.parts = clamp(4 * sms / cells, by_rows < 8 ? by_rows : 8);
    p.key_room = (int64_t)p.key_tiles * MT;
    p.lse_floats = ((size_t)st.T * H + 3) / 4 * 4;
    p.stat_floats = p.stat_parts > 1 ? ((size_t)st.T * H * p.stat_parts * 2 + 3) / 4 * 4 : 0;
    p.floats = p.lse_floats + p.stat_floats + (p.parts > 1 ? (size_t)p.parts * st.B * G * p.key_room : 0);
    return p;
}

bool weigh_tc_takes(const WeighArgs& w, bool four) {
    auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    return w.D <= 128 && w.D % 4 == 0 && w.ld % 4 == 0 && al(w.q) && (four || al(w.kpool));
}

int weigh_tc(const WeighArgs& w, const b200seq_step& st, const WeighTcPlan& p, float* scratch, bool four, cudaStream_t cs) {
    const int64_t g0 = (int64_t)p.tiles * w.G, g1 = (int64_t)p.key_tiles * p.parts * w.G * st.B;
    if (g0 > 0x7fffffff || g1 > 0x7fffffff) return fail(B200SEQ_ERR_UNSUPPORTED, "key_weights: too many tiles for one launch");
    TcArgs a = {};
    a.w = w, a.w.lse = scratch, a.stat = reinterpret_cast<float2*>(scratch + p.lse_floats), a.psum = scratch + p.lse_floats + p.stat_floats, a.stat_parts = p.stat_parts, a.key_room = p.key_room, a.B = st.B;
    a.parts = p.stat_parts, a.tiles = p.tiles;
    cudaError_t e = run<false>(a, st, dim3((unsigned)g0, 1, p.stat_parts), four, cs);
    if (e != cudaSuccess) return cuda_status(e, "key_weights");
    count_launch();
    if (p.stat_parts > 1) {
        launch_chained(weigh_lse_kernel, dim3((unsigned)(((int64_t)st.T * w.H + 127) / 128)), 128, 0, cs, a, st.T * w.H);
        SEQ_LAUNCH_CHECK("key_weights");
    }
    a.parts = p.parts, a.tiles = p.key_tiles;
    e = run<true>(a, st, dim3((unsigned)g1), four, cs);
    if (e != cudaSuccess) return cuda_status(e, "key_weights");
    count_launch();
    if (p.parts > 1) {
        launch_chained(weigh_parts_kernel, dim3((unsigned)((p.key_room + 255) / 256), w.G, st.B), 256, 0, cs, a, st);
        SEQ_LAUNCH_CHECK("key_weights");
    }
    return 0;
}

}  // namespace b200seq
