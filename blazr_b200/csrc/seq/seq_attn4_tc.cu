// seq_attn4_tc.cu -- the attend step of prompt portions over KV pages held in 4 bits, on the 5th-generation tensor cores.
//
// What the cache holds enters the products as it is: s (u - 8) is an f16 number (seq_kv4.cuh), and the m + 8 s of a row's groups are eight more values of it, as high and low
// f16 parts, against the group sums of q (keys), or as columns of their own (values).  Only q and the weights are rounded: to two f16 parts (22 bits) each where results are
// f32; to one (11 bits, off by up to 2^-11 of a value) where they are bf16, which is an eighth of what such a result itself and the bf16 activations behind q are rounded by;
// weights far below the row's largest keep as much of it as the kernel says.  So scores and sums of values are one or two products each where f32 operands (seq_attn_tc.cu)
// take six.
//
// One CTA works on rows of 128 (token, query head) pairs of one key head against tiles of 64 keys.  A soft-max warp's thread owns a row; two groups of four such warps alternate,
// one in the soft-max while the other's products are in the tensor pipe:
//   MT = 2        two row tiles, a group each (heads up to 64, rows for all SMs)
//   MT = 1, TG    one row tile, the groups take turns with the key tiles and are merged at the end
//   MT = 1        one group, whose consecutive key tiles alternate (heads above 64 with f32 results: no registers for two)
// The values of 64 keys leave the tensor core and are summed over the key tiles by rounded adds in registers; heads above 64 with bf16 results stay there (TA: the
// sums' truncation, 2^-24 of them a product, is nothing to such a result) and are rescaled when a row's maximum has grown by 2^5.
//   first 4 or 8 warps     soft-max: a row's maximum, sum and value sums stay in its thread's registers, nothing is shuffled
//   next 8 warps           loaders, four for keys and four for values: codes and parameters from the pages, a tile ahead, expanded into 128-byte swizzled rows.  Both lie
//                          alike, [key][value]: K-major for the scores, mn-major for the sums
//   last 4 warps           the first of them issues the MMAs
// The order of a row's values is that of its code words (pairs of fields that one AND takes out): q is permuted alike, results are put back in order as they are stored.
// Registers (setmaxnreg, per thread): launched with 96 (two groups) or 128 (one) for all; soft-max 160 / 240, loaders 64 / 104, issuer 32 / 64: the sums
// (2 * 160 + 2 * 64 + 32 = 5 * 96, 240 + 2 * 104 + 64 = 4 * 128) are what the block was launched with.
// Measured: 2048 tokens of 32 query heads of 8 key heads of 128, bf16 results: 79 us (435 TFLOP/s of what every row sees), f32 121; 531 tokens behind 5000, heads of 64, window 2048,
// f32: 40 us.  A CTA takes about 9 us beside its key tiles (queries into the tensor core's memory, the first tile's way through all roles, results out) and 0.7 a key tile, which
// the instructions of expanding and soft-max bound (tensor pipe active 20 %).
// Every wait is bounded (tc_pair.cuh): one that runs out sets bit 1 of the library's error flags and the CTA leaves through the common exit.
#include "seq_attn4.cuh"
#include "tc_split.cuh"

namespace b200seq {

namespace {

using namespace tcsplit;

constexpr int KT = 64;                       // keys per tile
constexpr int PLANE = KT * 128;              // bytes of one 64-key x 64-wide block
constexpr int SLOT_COLS = 64;                // scores f32 [64], then the weights' parts [32] [32] in the same columns
constexpr float LOG2E = 1.4426950408889634f;
constexpr float SLACK = 5.f;                  // TA: a row's reference is raised when a score passes it by this much (base 2: weights up to 2^5)

__host__ __device__ constexpr int blocks_of(int groups) { return (4 * groups + 9) / 8; }   // 16-byte pieces of a row: 4 a group, m + 8 s, zeros
__host__ __device__ constexpr int columns_of(int groups) { return 32 * groups + 16; }

__device__ __forceinline__ uint32_t h2(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ __half2 h2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t field_or(uint32_t x, uint32_t mask, uint32_t magic) {
    uint32_t w;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(w) : "r"(x), "r"(mask), "r"(magic));
    return w;
}
// a word's eight codes as eight f16 s (u - 8): pairs of fields (i, i + 4), i = 0 .. 3.  s: the steps of the word's low and high half.  A field in the mantissa of 1024 or of
// 64 is that number plus u; 8 and the number go first, exactly, then comes the step (72 s is no f16 number where s is large: no multiply-add).
__device__ __forceinline__ void expand(uint32_t w, __half2 s, uint32_t (&x)[4]) {
    const __half2 off = __floats2half2_rn(-1032.f, -1032.f), off64 = __floats2half2_rn(-72.f, -72.f);
    const uint32_t w8 = w >> 8;
    x[0] = h2(__hmul2_rn(__hadd2_rn(h2(field_or(w, 0x000F000Fu, 0x64006400u)), off), s));
    x[1] = h2(__hmul2_rn(__hadd2_rn(h2(field_or(w, 0x00F000F0u, 0x54005400u)), off64), s));
    x[2] = h2(__hmul2_rn(__hadd2_rn(h2(field_or(w8, 0x000F000Fu, 0x64006400u)), off), s));
    x[3] = h2(__hmul2_rn(__hadd2_rn(h2(field_or(w8, 0x00F000F0u, 0x54005400u)), off64), s));
}
// m + 8 s of two groups, as high and low f16 parts (the low one is what rounding the high one leaves: an f16 number)
__device__ __forceinline__ void centres(__half2 s, __half2 m, uint32_t& high, uint32_t& low) {
    const __half2 eight = __floats2half2_rn(8.f, 8.f), d = __hfma2(s, eight, m), t = __hsub2_rn(d, m);
    high = h2(d), low = h2(__hadd2_rn(__hsub2_rn(m, __hsub2_rn(d, t)), __hfma2(s, eight, __hneg2(t))));
}
__device__ __forceinline__ void sts16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void st1(uint32_t taddr, uint32_t r) { asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(r) : "memory"); }
__device__ __forceinline__ void ld8(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
// place of value d of a row in the order of its code words
__host__ __device__ constexpr int value_place(int d, int NV) {
    const int g = d >> 5, r = (d >> 2) & 7, i = d & 3;
    return NV == 1 ? (r >> 1) * 8 + 2 * i + (r & 1) : (g >> 1) * 64 + ((r & 1) * 4 + (r >> 1)) * 8 + 2 * i + (g & 1);
}

template <int N>
struct Codes {
    uint32_t w[N], p[N];
};
// a thread's quarter of a row's codes and the row's parameters
template <int N>
__device__ __forceinline__ void load_codes(Codes<N>& c, const uint8_t* w, const uint8_t* p, bool in) {
    if (!in) {
#pragma unroll
        for (int i = 0; i < N; ++i) c.w[i] = c.p[i] = 0;
    } else if (N == 4) {
        const uint4 a = *reinterpret_cast<const uint4*>(w), b = *reinterpret_cast<const uint4*>(p);
        c.w[0] = a.x, c.w[1 % N] = a.y, c.w[2 % N] = a.z, c.w[3 % N] = a.w, c.p[0] = b.x, c.p[1 % N] = b.y, c.p[2 % N] = b.z, c.p[3 % N] = b.w;
    } else if (N == 2) {
        const uint2 a = *reinterpret_cast<const uint2*>(w), b = *reinterpret_cast<const uint2*>(p);
        c.w[0] = a.x, c.w[1 % N] = a.y, c.p[0] = b.x, c.p[1 % N] = b.y;
    } else {
        c.w[0] = *reinterpret_cast<const uint32_t*>(w), c.p[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}
// Into shared memory: piece i of row `key` lies at block i / 8, place (i % 8) ^ (key % 8).  at: the row's first block; even, odd: where this thread's pieces `quarter` and
// quarter + 4 of a block lie in it (the same for all blocks, and for key + 8).
template <int N, bool KEY>
__device__ __forceinline__ void put_codes(const Codes<N>& c, uint32_t even, uint32_t odd) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        uint32_t x[4];
        __half2 s;
        uint32_t to;
        if (KEY) {            // words [part][group]: word i is group i of part `quarter`: piece 4 i + quarter
            s = __low2half2(h2(c.p[i])), to = ((i & 1) ? odd : even) + (i >> 1) * PLANE;
        } else if (N == 1) {  // two parts of the one group: piece `quarter`
            s = __low2half2(h2(c.p[0])), to = even;
        } else {              // 16-bit words [part][group]: word i is two groups of part 2 quarter + r: piece 8 gp + 4 r + quarter
            const int gp = N == 4 ? i & 1 : 0, r = N == 4 ? i >> 1 : i;
            s = __lows2half2(h2(c.p[2 * gp]), h2(c.p[(2 * gp + 1) % N])), to = (r ? odd : even) + gp * PLANE;
        }
        expand(c.w[i], s, x);
        sts16(to, x[0], x[1], x[2], x[3]);
    }
}
// group `quarter`'s m + 8 s of two keys into their rows' piece 4 N: four high parts, four low parts
template <int N>
__device__ __forceinline__ void put_centres(const Codes<N>& c0, const Codes<N>& c1, int quarter, uint32_t at0, uint32_t at1) {
    auto pick = [&](const Codes<N>& c) {
        uint32_t p = c.p[0];
        if (N > 1) p = quarter & 1 ? c.p[1 % N] : p;
        if (N == 4) p = quarter & 2 ? (quarter & 1 ? c.p[3 % N] : c.p[2 % N]) : p;
        return quarter < N ? p : 0u;
    };
    const uint32_t a = pick(c0), b = pick(c1);
    uint32_t hi, lo;
    centres(__lows2half2(h2(a), h2(b)), __highs2half2(h2(a), h2(b)), hi, lo);
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at0), "h"((uint16_t)hi) : "memory");
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at1), "h"((uint16_t)(hi >> 16)) : "memory");
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at0 + 8), "h"((uint16_t)lo) : "memory");
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at1 + 8), "h"((uint16_t)(lo >> 16)) : "memory");
}

// The key tiles of one pool, expanded into their stages: four warps, four threads a key, two keys a thread.  A tile's codes are asked for while the tile before it is
// expanded, its pages a tile earlier.  stage: of tile 0 (tile 1's is `pitch` bytes on); full, free: the stages' barriers.
template <int N, bool KEY>
__device__ __forceinline__ void load_tiles(const uint8_t* pool, const int32_t* bt, int bs, int g, int G, const KeySpan<KT>& span, int split, int parts, int ntile, int hi, uint32_t stage,
                                           uint32_t pitch, uint32_t full, uint32_t free, int lw, int lane, volatile int* ab, int* err) {
    // eight lanes store pieces of keys k and k + 4: their places in the swizzle fill a 128-byte line
    const int j8 = lane >> 2, key = lw * 16 + ((j8 & 1) << 2) + (j8 >> 1), quarter = lane & 3;
    if (quarter == 0) {   // the pieces behind m + 8 s stay zero
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int k = key + 8 * u;
                sts16(stage + s * pitch + k * 128 + ((4 * N + 1) >> 3) * PLANE + ((((4 * N + 1) & 7) ^ (k & 7)) << 4), 0, 0, 0, 0);
            }
    }
    uint32_t even = stage + key * 128 + ((quarter ^ (key & 7)) << 4), odd = stage + key * 128 + (((4 + quarter) ^ (key & 7)) << 4);
    uint32_t centre = stage + key * 128 + ((4 * N) >> 3) * PLANE + ((((4 * N) & 7) ^ (key & 7)) << 4) + 2 * quarter;
    // Pages of 16: a tile's 64 keys are four whole pages, and a thread's keys (key and key + 8) lie at fixed places of one of them.  Other sizes: each key is looked up.
    const bool whole = bs == 16;
    const Kv4Row r0 = kv4_row(0, key & 15, 16, g, G, N), r1 = kv4_row(0, (key & 15) + 8, 16, g, G, N);      // (key % 16 < 8)
    const uint8_t *w0 = pool + r0.codes + 4 * N * quarter, *p0 = pool + r0.params;
    const uint32_t pitch_w = (uint32_t)(r1.codes - r0.codes), pitch_p = (uint32_t)(r1.params - r0.params), page_bytes = (uint32_t)G * (16 * N * 20);
    int page[2] = {0, 0}, pos = 0;
    auto lookup = [&](int j) {
        pos = span.key0(split + j * parts) + key;
        if (whole) {
            if (pos <= hi) page[0] = bt[pos >> 4];
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) page[u] = bt[min(pos + 8 * u, hi) / bs];
        }
    };
    Codes<N> next[2];
    auto fetch = [&]() {   // the tile that was looked up
        if (whole) {
            const uint64_t at = (uint64_t)(uint32_t)kv4_page_read(page[0], err) * page_bytes;
            load_codes<N>(next[0], w0 + at, p0 + at, pos <= hi), load_codes<N>(next[1], w0 + at + pitch_w, p0 + at + pitch_p, pos + 8 <= hi);
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int kp = min(pos + 8 * u, hi);
                const Kv4Row at = kv4_row(kv4_page_read(page[u], err), kp % bs, bs, g, G, N);
                load_codes<N>(next[u], pool + at.codes + 4 * N * quarter, pool + at.params, pos + 8 * u <= hi);
            }
        }
    };
    if (ntile > 0) {
        lookup(0);
        fetch();
        if (ntile > 1) lookup(1);
    }
    uint32_t there = pitch;
#pragma unroll 1
    for (int j = 0; j < ntile; ++j) {
        const int s = j & 1;
        const Codes<N> c0 = next[0], c1 = next[1];
        if (j + 1 < ntile) {
            fetch();
            if (j + 2 < ntile) lookup(j + 2);
        }
        if (!bar_wait<false>(free + 8 * s, ((j >> 1) & 1) ^ 1, ab)) return;
        put_codes<N, KEY>(c0, even, odd);
        put_codes<N, KEY>(c1, even + 1024, odd + 1024);
        put_centres<N>(c0, c1, quarter, centre, centre + 1024);
        async_fence();
        __syncwarp();
        if (lane == 0) bar_arrive(full + 8 * s);
        even += there, odd += there, centre += there, there = 0u - there;      // the other stage
    }
}

// MT row tiles; TG: two groups on one; NK, NV groups of 32 of a key and a value; NP parts of q and of a weight; CAP: scores are soft-capped
template <int MT, bool TG, int NK, int NV, int NP, bool CAP>
__global__ void __launch_bounds__((4 * (TG ? 2 : MT) + 12) * 32, 1) attn4_tc_kernel(const __grid_constant__ Attn4Args a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_base;
    __shared__ int abort_sh;
    __shared__ __align__(8) uint64_t bars[16];
    __shared__ float row_factor[TG ? 128 : 1];
    static_assert(!(TG && MT == 2) && (NV < 4 || (MT == 1 && (!TG || NP == 1))), "");
    constexpr bool TA = TG && NV == 4;                 // value sums stay in TMEM
    // Weights become f16 parts times a power of two: up to 2^15, so that they are off by 2^-40 (TA: 2^-35) of the row's largest at most however small they are (f16 numbers end
    // at 2^-24).  One part: the exponent takes the power in, which rounds it at up to 2^4 (2^-21).  Two: that would show (f32 results, 600 tokens of heads of 64: rms error
    // 4.3e-8, multiplied 3.1e-8; 26.2 us, 27.0).  TA, slack 2 instead of 5: references are raised, and sums in TMEM rescaled, too often (2048 tokens 88 us, 79).
    constexpr float SHIFT = TA ? 10.f : 15.f, UP = TA ? 0x1p10f : 0x1p15f, DOWN = 1.f / UP;
    constexpr int GROUPS = TG ? 2 : MT, SW = 4 * GROUPS;   // soft-max warps
    constexpr int KBYTES = blocks_of(NK) * PLANE, VBYTES = blocks_of(NV) * PLANE, STAGE = KBYTES + VBYTES, VM = 32 * NV, OCOLS = columns_of(NV), QP = columns_of(NK) / 2;
    constexpr int PITCH = 32 * (NK > NV ? NK : NV) + 4, RL = 8 * NK;   // floats of a staged row (16-byte pieces of a warp's rows in different banks); lanes a row of q takes
    const uint32_t kv = (sa(smem_raw) + 1023u) & ~1023u;
    float* const stage_rows = reinterpret_cast<float*>(smem_raw + (kv - sa(smem_raw)) + 2 * STAGE);   // [128 MT][PITCH]: q on the way in, results on the way out
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;   // warp-uniform: the roles branch on it
    const int D = a.D, V = a.V, H = a.H, G = a.G;
    const uint32_t B0 = sa(bars);
    const uint32_t k_full = B0, k_free = B0 + 16, v_full = B0 + 32, v_free = B0 + 48, s_full = B0 + 64, p_ready = B0 + 80, o_full = B0 + 96;
    volatile int* ab = &abort_sh;
    int e, t0, nq;
    // the tiles with the most keys first, for all heads at once, so that the last CTAs to start are short
    const int units = G * a.HB, n = (int)gridDim.x / units, ord = (int)blockIdx.x / units, unit = (int)blockIdx.x - ord * units;
    int tile_no = n - 1 - ord;
    if (a.chunk > 0 && a.chunk % a.QT == 0 && a.chunk / a.QT < n) {   // (in a step of chunks those are the last ones of every chunk)
        const int per = a.chunk / a.QT, nc = (n + per - 1) / per, rem = n - (nc - 1) * per, longer = (per - rem) * (nc - 1);
        if (ord < longer) tile_no = (ord % (nc - 1)) * per + per - 1 - ord / (nc - 1);
        else tile_no = ((ord - longer) % nc) * per + rem - 1 - (ord - longer) / nc;
    }
    if (st.B == 1) {
        e = 0, t0 = tile_no * a.QT, nq = min(a.QT, min(st.T, st.ent_start[1]) - t0);
        if (nq <= 0) return;
    } else if (!attn_find_tile(st, tile_no, a.QT, e, t0, nq)) return;
    const int p0 = st.tok_pos[t0];
    const int g = unit / a.HB, hb = unit - g * a.HB, R = H / G;
    const int h0 = g * R + hb * a.Rb, nh = min(a.Rb, R - hb * a.Rb);
    const int split = blockIdx.z;
    {   // the queries' rows on their way while the rest is set up: whole rows at a time (read by their threads they cost a 128-byte line a lane and load), by all warps
        constexpr int WARPS = SW + 12, STEP = WARPS * (32 / RL);
        const int d4 = 4 * (lane & (RL - 1));
        const float* qrow = a.q + (int64_t)t0 * a.ld + (int64_t)h0 * D + d4;
        const uint32_t to = sa(stage_rows) + d4 * 4;
#pragma unroll 2
        for (int row = warp * (32 / RL) + lane / RL; row < 128 * MT; row += STEP) {
            const int rt = row / a.Rb, rh = row - rt * a.Rb;
            const bool in = rt < nq && rh < nh && d4 < D;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + row * PITCH * 4), "l"(in ? qrow + (int64_t)rt * a.ld + rh * D : a.q), "r"(in ? 16 : 0)
                         : "memory");                  // (nothing is read where there is no row; its place becomes zero)
        }
    }
    const int hi = p0 + nq - 1, bs = st.block_size;
    const int32_t* bt = st.block_table + (int64_t)e * st.max_blocks;
    if (p0 < 0 || hi / bs >= st.max_blocks) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (threadIdx.x == 0) atomicOr(a.err, 1);
        if (a.parts > 1)                              // (a sum below zero: no parts of these rows)
            for (int i = threadIdx.x; i < nq * nh; i += blockDim.x) a.part[(((int64_t)(t0 + i / nh) * H + h0 + i % nh) * a.parts + split) * (V + 4) + 1] = -1.f;
        return;
    }
    const KeySpan<KT> span(a, p0, hi);
    const int ntile = span.total > split ? (span.total - split + a.parts - 1) / a.parts : 0;   // tiles split, split + parts, ...
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(k_full + 8 * i, 4), bar_init(k_free + 8 * i, 1), bar_init(v_full + 8 * i, 4), bar_init(v_free + 8 * i, 1);
            bar_init(s_full + 8 * i, 1), bar_init(p_ready + 8 * i, 4), bar_init(o_full + 8 * i, 1);
        }
        bar_init(B0 + 112, 1);
        abort_sh = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(sa(&tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base;
    const uint32_t slot0 = tmem, o0 = tmem + 2 * SLOT_COLS, q0 = o0 + GROUPS * OCOLS;   // columns: slots | value tiles | query parts

    if (warp < SW) {
        // ===================== soft-max: thread == row =====================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(GROUPS == 2 ? 160 : 240));
        const int m = warp >> 2, q = warp & 3;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const int r = (TG ? 0 : m * 128) + q * 32 + lane;
        const int tq = r / a.Rb, hr = r - tq * a.Rb;
        const bool live = tq < nq && hr < nh;
        int rlo = 0, rhi = 0x3fffffff;   // rows without a token see everything and are not stored
        const int keep = a.window > 0 ? a.keep_first : 0;
        float factor = a.scale;
        if (live) {
            const RowSpan rs(a, p0 + tq);
            rlo = rs.lo, rhi = rs.p;
            if (a.head_scale) factor *= a.head_scale[h0 + hr];
        }
        // soft-max in base 2 over raw scores: weight = 2^(c s - mb), mb = c max(s); the sign of the factor and a power of two go into the query.  With a soft cap the
        // scores are scaled and capped first (CAP) and c is 1.
        float zf = 0.f;
        float* const mine_row = stage_rows + r * PITCH;
        constexpr bool SPLIT = TG && NK == 4;     // both groups: two of the four groups of 32 each
        if (!TG || SPLIT || m == 0) {   // this row's query, in the order of the code words, and its group sums, to TMEM
            const float* src = mine_row;
            float top = 0.f;
#pragma unroll 8
            for (int d = 0; d < 32 * NK; d += 4) {
                const float4 x = ld4(src + d);
                top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
            }
            const int ex = (int)(__float_as_uint(top) >> 23);
            const bool norm = ex >= 20 && ex < 255;     // the largest into [2^4, 2^5); a row of zeros, denormals or infinities as it is
            const float up = copysignf(norm ? __uint_as_float((uint32_t)(254 - ex + 4) << 23) : 1.f, factor), down = norm ? __uint_as_float((uint32_t)(ex - 4) << 23) : 1.f;
            zf = fmaxf(fabsf(factor) * down * (CAP ? 1.f : LOG2E), 1e-37f);
            const uint32_t qa = q0 + lanes + (TG ? 0 : m * NP * QP);
            float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k_ = 0; k_ < (SPLIT ? 2 : NK); ++k_) {
                const int k = SPLIT ? 2 * m + k_ : k_;
#pragma unroll 1
                for (int c2 = 0; c2 < 4; c2 += 2) {
                    uint32_t ph[8], pl[8];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int d = 32 * k + 8 * (c2 + u);
                        const float4 x = ld4(src + d), y = ld4(src + d + 4);     // (zeros behind D)
                        const float f[8] = {x.x * up, x.y * up, x.z * up, x.w * up, y.x * up, y.y * up, y.z * up, y.w * up};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const __half2 h = __floats2half2_rn(f[i], f[i + 4]);
                            const float2 b = __half22float2(h);
                            ph[4 * u + i] = h2(h), pl[4 * u + i] = h2(__floats2half2_rn(f[i] - b.x, f[i + 4] - b.y));
                            sums[k_] += f[i] + f[i + 4];
                        }
                    }
                    st8(qa + (4 * k + c2) * 4, ph);
                    if (NP == 2) st8(qa + QP + (4 * k + c2) * 4, pl);
                }
            }
            // the sums of q, two groups a column, against the high and the low parts of m + 8 s
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (SPLIT && i) break;
                const __half2 h = __floats2half2_rn(sums[2 * i], sums[2 * i + 1]);
                const float2 b = __half22float2(h);
                const uint32_t hi2 = h2(h), lo2 = h2(__floats2half2_rn(sums[2 * i] - b.x, sums[2 * i + 1] - b.y)), at = qa + 16 * NK + (SPLIT ? m : i);
                st1(at, hi2), st1(at + 2, hi2);
                if (NP == 2) st1(at + QP, lo2), st1(at + QP + 2, lo2);
            }
            if (!SPLIT || m == 0) {
#pragma unroll
                for (int i = 4; i < 8; ++i) {
                    st1(qa + 16 * NK + i, 0u);
                    if (NP == 2) st1(qa + QP + 16 * NK + i, 0u);
                }
            }
            if (TG && !SPLIT) row_factor[q * 32 + lane] = zf;
            st_wait();
            fence_before();
        }
        asm volatile("bar.sync 1, %0;" ::"n"((SW + 1) * 32) : "memory");   // the queries are in place (with the MMA warp)
        if (TG && !SPLIT && m) zf = row_factor[q * 32 + lane];
        const float c = CAP ? 1.f : zf;
        const uint64_t cc = pk(c, c);
        float mx = -INFINITY, mb = -INFINITY, l = 0.f, rest[4] = {0.f, 0.f, 0.f, 0.f};
        constexpr int NACC = TA ? 1 : VM / 2;
        uint64_t acc[NACC];
#pragma unroll
        for (int i = 0; i < NACC; ++i) acc[i] = 0;
        bool ok = true;
        auto add_values = [&](int step) {   // acc += the value tile of a step
            ok = __all_sync(0xffffffffu, bar_wait<false>(o_full + 8 * (step & 1), (step >> 1) & 1, ab));
            if (!ok) return false;
            fence_after();
#pragma unroll
            for (int i = 0; i < VM; i += 32) {
                float o[32];
                ld32(o0 + lanes + m * OCOLS + i, o);
                ld_wait();
#pragma unroll
                for (int u = 0; u < 32; u += 2) acc[TA ? 0 : (i + u) >> 1] = add2(acc[TA ? 0 : (i + u) >> 1], pk(o[u], o[u + 1]));
            }
            float o[8];
            ld8(o0 + lanes + m * OCOLS + VM, o);
            ld_wait();
#pragma unroll
            for (int u = 0; u < 4; ++u) rest[u] += o[u] + o[4 + u];
            fence_before();
            return true;
        };
#pragma unroll 1
        for (int j = TG ? m : 0; j < ntile && ok; j += TG ? 2 : 1) {
            const int step = TG ? j : j * MT + m, slot = step & 1;
            const int k0 = span.key0(split + j * a.parts);
            const int lo = rlo - k0, hi1 = rhi + 1 - k0, kp = keep - k0;   // visible keys of this row, relative to the tile: [lo, hi1) and those below kp
            const bool whole = __all_sync(0xffffffffu, lo <= 0 && hi1 >= KT);
            const uint32_t S = slot0 + lanes + slot * SLOT_COLS;
            ok = __all_sync(0xffffffffu, bar_wait<false>(s_full + 8 * slot, (step >> 1) & 1, ab));   // (tcgen05 loads are the whole warp's)
            if (!ok) break;
            fence_after();
            float v[KT];
            ld32(S, v);
            ld32(S + 32, v + 32);
            ld_wait();
            if (CAP) {
#pragma unroll
                for (int i = 0; i < KT; ++i) v[i] = a.softcap * LOG2E * tanhf(v[i] * zf / a.softcap);
            }
            if (!whole) {
                auto below = [](int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); };
                const uint32_t s0 = below(hi1) & (~below(lo) | below(kp)), s1 = below(hi1 - 32) & (~below(lo - 32) | below(kp - 32));
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    v[i] = (s0 >> i) & 1u ? v[i] : -INFINITY;
                    v[32 + i] = (s1 >> i) & 1u ? v[32 + i] : -INFINITY;
                }
            }
            float m0 = fmaxf(v[0], v[1]), m1 = fmaxf(v[2], v[3]);
#pragma unroll
            for (int i = 4; i < KT; i += 4) m0 = fmaxf(m0, fmaxf(v[i], v[i + 1])), m1 = fmaxf(m1, fmaxf(v[i + 2], v[i + 3]));
            const float tmax = fmaxf(m0, m1);
            float corr = 1.f;
            // (rounded so that no exponent below exceeds SLACK or 0, however large the scores: the weights' f16 parts end there)
            if (!TA || __fmul_ru(tmax, c) > __fadd_rd(mb, SLACK)) {      // (TA: a row's reference stays until a score passes it by SLACK)
                mx = fmaxf(mx, tmax);
                const float mbn = __fmul_ru(mx, c);
                corr = mx == -INFINITY ? 1.f : ex2(mb - mbn);   // 0 at the first visible key
                mb = mbn;
            }
            const float off = mx == -INFINITY ? 0.f : (NP == 1 ? __fsub_rd(SHIFT, mb) : -mb);
            const uint64_t off2 = pk(off, off);
            uint64_t sum = 0;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {   // the weights' parts (over the scores, which are in registers)
                uint32_t ph[8], pl[8];
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    float x, y;
                    upk(fma2(pk(v[16 * q4 + i], v[16 * q4 + i + 1]), cc, off2), x, y);
                    x = ex2(x), y = ex2(y);
                    sum = add2(sum, pk(x, y));
                    if (NP == 2) upk(mul2(pk(x, y), pk(UP, UP)), x, y);
                    const __half2 h = __floats2half2_rn(x, y);
                    ph[i >> 1] = h2(h);
                    if (NP == 2) {
                        const float2 b = __half22float2(h);
                        pl[i >> 1] = h2(__floats2half2_rn(x - b.x, y - b.y));
                    }
                }
                st8(S + 8 * q4, ph);
                if (NP == 2) st8(S + 32 + 8 * q4, pl);
            }
            float sx, sy;
            upk(sum, sx, sy);
            l = fmaf(l, corr, sx + sy);
            const uint64_t corr2 = pk(corr, corr);
            const bool same = __all_sync(0xffffffffu, corr == 1.f);
            // one group: the value tile of the key tile before, whose product ran beside this soft-max
            if (GROUPS == 1 && j > 0 && !add_values(step - 1)) break;
            if (!same && !TA) {
#pragma unroll
                for (int i = 0; i < NACC; ++i) acc[i] = mul2(acc[i], corr2);
#pragma unroll
                for (int i = 0; i < 4; ++i) rest[i] *= corr;
            }
            if (!same && TA && j >= 2) {        // behind the product of this group's tile before
                ok = __all_sync(0xffffffffu, bar_wait<false>(o_full + 8 * slot, ((step >> 1) & 1) ^ 1, ab));
                if (!ok) break;
                fence_after();
                const uint32_t O = o0 + lanes + m * OCOLS;
#pragma unroll 1
                for (int i = 0; i < OCOLS; i += 16) {
                    float o[16];
                    ld16(O + i, o);
                    ld_wait();
                    uint32_t u[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(o[k] * corr);
                    st8(O + i, u), st8(O + i + 8, u + 8);
                }
            }
            st_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(p_ready + 8 * slot);
            // two groups: this key tile's, while the next scores are made (the other group keeps the tensor pipe busy)
            if (GROUPS == 2 && !TA && !add_values(step)) break;
        }
        if (NP == 1) l *= DOWN;                    // (the values' sums are taken down as results are made)
        if (GROUPS == 1 && ok && ntile > 0) add_values(ntile - 1);
        const int mine = TG ? (ntile - m + 1) / 2 : ntile;    // key tiles of this group
        if (TA && ok && mine > 0) {
            const int last = 2 * (mine - 1) + m;
            ok = __all_sync(0xffffffffu, bar_wait<false>(o_full + 8 * (last & 1), (last >> 1) & 1, ab));
            fence_after();
        }
        // value sums of 32 columns, from registers or TMEM
        auto values = [&](int i, float (&o)[32]) {
            if (TA) {
                if (mine > 0) {
                    ld32(o0 + lanes + m * OCOLS + i, o);
                    ld_wait();
                } else {
#pragma unroll
                    for (int u = 0; u < 32; ++u) o[u] = 0.f;
                }
            } else {
#pragma unroll
                for (int u = 0; u < 32; u += 2) upk(acc[TA ? 0 : (i + u) >> 1], o[u], o[u + 1]);
            }
        };
        if (TA && ok && mine > 0) {
            float o[8];
            ld8(o0 + lanes + m * OCOLS + VM, o);
            ld_wait();
#pragma unroll
            for (int u = 0; u < 4; ++u) rest[u] = o[u] + o[4 + u];
        }
        // Two groups on one row tile are merged through shared memory, over the key and value stages (all that was issued has been waited for by both): each gives the
        // other its share of the columns, a block of 64 where there are two, all to the first one where there is one.
        constexpr int W = VM < 64 ? VM : 64, XP = W + 7;    // (odd: a warp's rows lie in different banks)
        const int keep_block = NV == 4 && TG ? m : 0;
        float f0 = 1.f, f1 = 0.f;
        const float* other = nullptr;
        if (TG) {
            float* const base = reinterpret_cast<float*>(smem_raw + (kv - sa(smem_raw)));
            constexpr int XQ = NV == 4 ? XP : 8;            // (one block of columns: the first group gives its maximum and sums alone)
            static_assert(128 * (XP + XQ) * 4 <= 2 * STAGE, "the stages hold both groups' parts");
            float *const second = base + (q * 32 + lane) * XP, *const first = base + 128 * XP + (q * 32 + lane) * XQ;
            float* const x = m ? second : first;
            const float* const y = m ? first : second;
            asm volatile("bar.sync 2, %0;" ::"n"(SW * 32) : "memory");
            x[0] = mb, x[1] = l;
#pragma unroll
            for (int u = 0; u < 4; ++u) x[2 + u] = rest[u];
            if (NV == 4 || m == 1) {
#pragma unroll
                for (int i = 0; i < W; i += 32) {
                    float o[32];
                    values(NV == 4 ? (m ? i : 64 + i) : i, o);
#pragma unroll
                    for (int u = 0; u < 32; ++u) x[6 + i + u] = o[u];
                }
            }
            asm volatile("bar.sync 2, %0;" ::"n"(SW * 32) : "memory");
            const float mb1 = y[0], l1 = y[1], top = fmaxf(mb, mb1);
            f0 = l == 0.f ? 0.f : ex2(mb - top), f1 = l1 == 0.f ? 0.f : ex2(mb1 - top);    // (0: no key that the row sees)
            l = m ? fmaf(l1, f1, l * f0) : fmaf(l, f0, l1 * f1), mb = top;                 // (the first group's first: the same sum in both)
#pragma unroll
            for (int u = 0; u < 4; ++u) rest[u] = fmaf(rest[u], f0, y[2 + u] * f1);
            other = y + 6;
        }
        if (ok) {   // (all lanes: TMEM is read by whole warps)
            const int t = t0 + tq, h = h0 + hr;
            float f = DOWN;
            if (live && a.parts == 1) {
                float gate = 1.f, den = l, resc = 1.f;
                if (a.gated && !a.gate_elem) gate = sigmoidf_acc(a.gate[(int64_t)t * a.gld + h]);
                if (a.sink) {   // the sink's term, under the larger of the two maxima
                    const float sk = a.sink[h] * LOG2E, top = fmaxf(mb, sk);
                    resc = ex2(mb - top);
                    den = fmaf(l, resc, ex2(sk - top));
                }
                f = gate * resc / den * DOWN;
            } else if (live && (!TG || m == 0)) {
                float* pp = a.part + (((int64_t)t * H + h) * a.parts + split) * (V + 4);
                pp[0] = mb, pp[1] = l;
            }
            // blocks of 64 columns in the order of the code words are the values of two groups (32 columns: of the one group); through shared memory, so that rows are
            // stored whole
#pragma unroll
            for (int b = 0; b < (NV == 4 && !TG ? 2 : 1); ++b) {
                if (TG && NV < 4 && m) break;
                const int i0 = NV == 4 && TG ? 64 * keep_block : 64 * b;
                float o[W];
                __syncwarp();
                values(i0, *reinterpret_cast<float(*)[32]>(o));
                if (W == 64) values(i0 + 32, *reinterpret_cast<float(*)[32]>(o + W - 32));
                if (TG) {
#pragma unroll
                    for (int u = 0; u < W; ++u) o[u] = f1 != 0.f || f1 != f1 ? fmaf(other[u], f1, o[u] * f0) : o[u] * f0;
                }
                const float r0 = NV == 4 && i0 ? rest[2] : rest[0], r1 = NV == 4 && i0 ? rest[3] : rest[1];
#pragma unroll
                for (int d = 0; d < W; d += 4) {
                    float y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = (o[value_place(d + i, W == 64 ? 2 : 1)] + (d < 32 ? r0 : r1)) * f;
                    *reinterpret_cast<float4*>(mine_row + i0 + d) = make_float4(y[0], y[1], y[2], y[3]);
                }
            }
        }
        if (TG) asm volatile("bar.sync 2, %0;" ::"n"(SW * 32) : "memory");      // both groups store rows, half of them each
        __syncwarp();
        if (ok) {
            const bool wide = (V & 3) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
            constexpr int MINE = TG ? 16 : 32;
            const int row0 = TG ? q * 32 + 16 * m : m * 128 + q * 32;
            int rt = row0 / a.Rb, rh = row0 - rt * a.Rb;
            auto each = [&](auto&& store) {     // this warp's rows: store(row in shared memory, its number among all (token, head) pairs)
#pragma unroll 4
                for (int i = 0; i < MINE; ++i) {
                    if (rt < nq && rh < nh) store(stage_rows + (row0 + i) * PITCH, (int64_t)(t0 + rt) * H + h0 + rh);
                    if (++rh == a.Rb) rh = 0, ++rt;
                }
            };
            if (a.parts > 1) {
                each([&](const float* y, int64_t at) {
                    for (int d = lane; d < V; d += 32) a.part[(at * a.parts + split) * (V + 4) + 4 + d] = y[d];
                });
            } else if (wide && !a.gate_elem) {
                const bool in = 4 * lane < V;
                if (a.out_dtype == B200SEQ_F32) each([&](const float* y, int64_t at) { if (in) store_act4(a.out, B200SEQ_F32, at * V + 4 * lane, ld4(y + 4 * lane)); });
                else each([&](const float* y, int64_t at) { if (in) store_act4(a.out, B200SEQ_BF16, at * V + 4 * lane, ld4(y + 4 * lane)); });
            } else {
                each([&](const float* y, int64_t at) {
                    for (int d = lane; d < V; d += 32) store_act(a.out, a.out_dtype, at * V + d, y[d] * (a.gate_elem ? sigmoidf_acc(a.gate[at / H * a.gld + at % H * V + d]) : 1.f));
                });
            }
        }
    } else if (warp < SW + 8) {
        // ===================== loaders: four warps for keys, four for values =====================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(GROUPS == 2 ? 64 : 104));
        const int lw = warp - SW;
        if (lw < 4) load_tiles<NK, true>(a.kpool, bt, bs, g, G, span, split, a.parts, ntile, hi, kv, STAGE, k_full, k_free, lw, lane, ab, a.err);
        else load_tiles<NV, false>(a.vpool, bt, bs, g / a.vdiv, G / a.vdiv, span, split, a.parts, ntile, hi, kv + KBYTES, STAGE, v_full, v_free, lw - 4, lane, ab, a.err);
    } else {
        // ===================== MMA issuer =====================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(GROUPS == 2 ? 32 : 64));
        if (warp == SW + 8) asm volatile("bar.sync 1, %0;" ::"n"((SW + 1) * 32) : "memory");
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        if (warp == SW + 8 && elect()) {
            fence_after();
            constexpr uint32_t ids = (1u << 4) | ((uint32_t)(KT >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);                  // f16 x f16 -> f32
            constexpr uint32_t ido = (1u << 4) | (1u << 16) | ((uint32_t)(OCOLS >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);   // B is mn-major
            constexpr uint32_t O0 = 2 * SLOT_COLS, Q0 = O0 + GROUPS * OCOLS;
            const int steps = ntile * MT;
            bool ok = true;
            auto scores = [&](int step) {
                const int j = step / MT, s = j & 1, slot = step & 1, m = MT == 2 ? slot : 0;
                ok = bar_wait<false>(k_full + 8 * s, (j >> 1) & 1, ab);
                if (!ok) return;
                fence_after();
                const uint64_t kb = desc_k128(kv + s * STAGE);
                const uint32_t d = tm + slot * SLOT_COLS, qa = tm + Q0 + m * NP * QP;
#pragma unroll
                for (int pr = NP - 1; pr >= 0; --pr)     // the low parts of q first
#pragma unroll
                    for (int kk = 0; kk < 2 * NK + 1; ++kk)
                        mma_ts(d, qa + pr * QP + kk * 8, kb + (uint64_t)(((kk >> 2) * PLANE) / 16 + 2 * (kk & 3)), ids, (pr < NP - 1 || kk) ? 1u : 0u);
                commit_one(s_full + 8 * slot);
                if ((MT == 1 || slot == 1) && j + 2 < ntile) commit_one(k_free + 8 * s);   // (nobody waits for the last ones)
            };
            if (steps > 0) scores(0);
#pragma unroll 1
            for (int step = 0; step < steps && ok; ++step) {
                if (step + 1 < steps) {
                    if (step >= 1) ok = bar_wait<false>(o_full + 8 * ((step + 1) & 1), ((step - 1) >> 1) & 1, ab);   // the other slot's weights have been read
                    if (ok) scores(step + 1);
                    if (!ok) break;
                }
                const int j = step / MT, s = j & 1, slot = step & 1, m = GROUPS == 2 ? slot : 0;
                const uint32_t more = TA && j >= 2 ? 1u : 0u;          // on top of what is there
                ok = bar_wait<false>(v_full + 8 * s, (j >> 1) & 1, ab) && bar_wait<false>(p_ready + 8 * slot, (step >> 1) & 1, ab);
                if (!ok) break;
                fence_after();
                const uint64_t vb = desc_mn128(kv + s * STAGE + KBYTES, PLANE);
                const uint32_t d = tm + O0 + m * OCOLS, pa = tm + slot * SLOT_COLS;
#pragma unroll
                for (int pr = NP - 1; pr >= 0; --pr)
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
                        mma_ts(d, pa + 32 * pr + 8 * kk, vb + (uint64_t)(kk * 2048 / 16), ido, (pr < NP - 1 || kk) ? 1u : more);
                commit_one(o_full + 8 * slot);
                if ((MT == 1 || slot == 1) && j + 2 < ntile) commit_one(v_free + 8 * s);
            }
            if (!ok) {   // what was issued reads shared memory and TMEM: wait for it (bounded) before the CTA goes
                commit_one(B0 + 112);
                const unsigned long long t0_ = now_ns();
                while (!bar_try<false>(B0 + 112, 0) && now_ns() - t0_ < WAIT_NS) {}
            }
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && abort_sh) atomicOr(a.err, 2);
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int MT, bool TG, int NK, int NV, int NP, bool CAP>
cudaError_t run_one(const Attn4Args& a, const b200seq_step& st, dim3 grid, cudaStream_t cs) {
    constexpr int need = 2 * (blocks_of(NK) + blocks_of(NV)) * PLANE + 128 * MT * (32 * (NK > NV ? NK : NV) + 4) * 4 + 1024, smem = need < 120 * 1024 ? 120 * 1024 : need;   // one CTA per SM: it takes all of TMEM
    const auto kernel = attn4_tc_kernel<MT, TG, NK, NV, NP, CAP>;
    static bool ready[16] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 16 || !ready[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 16) ready[dev] = true;
    }
    launch_chained(kernel, grid, (4 * (TG ? 2 : MT) + 12) * 32, smem, cs, a, st);
    return cudaGetLastError();
}
template <int MT, int NK, int NV>
cudaError_t run(const Attn4Args& a, const b200seq_step& st, dim3 grid, cudaStream_t cs) {
    constexpr bool two = MT == 1;   // two groups on one row tile: not with f32 results of heads above 64
    if (a.softcap > 0.f) return a.out_dtype == B200SEQ_F32 ? run_one<MT, two && NV < 4, NK, NV, 2, true>(a, st, grid, cs) : run_one<MT, two, NK, NV, 1, true>(a, st, grid, cs);
    return a.out_dtype == B200SEQ_F32 ? run_one<MT, two && NV < 4, NK, NV, 2, false>(a, st, grid, cs) : run_one<MT, two, NK, NV, 1, false>(a, st, grid, cs);
}

}  // namespace

// What this kernel can do: whole 16-byte pieces of queries (the caller looks at addresses), keys and values of as many groups.
bool attn4_tc_takes(int D, int V) { return D % 8 == 0 && kv4_groups(D) == kv4_groups(V); }

// row tiles of 128 (256: two per CTA, heads of up to 64 and rows enough for all SMs)
Attn4TcPlan attn4_tc_plan(const b200seq_step& st, int H, int G, int D, int V, int64_t keys) {
    Attn4TcPlan p;
    const int R = H / G;
    p.mt = D <= 64 && V <= 64 && (int64_t)st.T * H >= 256ll * 148 ? 2 : 1;
    const int RQ = 128 * p.mt;
    p.Rb = R < RQ ? R : RQ, p.HB = (R + p.Rb - 1) / p.Rb, p.QT = RQ / p.Rb;
    p.tiles = ((int64_t)st.T + p.QT - 1) / p.QT + st.B - (st.B == 1);   // upper bound of the step's query tiles (exact for one entry)
    const int64_t each = (st.T + st.B - 1) / st.B;
    p.real = (int64_t)st.B * ((each + p.QT - 1) / p.QT) * G * p.HB;      // row tiles, were all entries equally long
    p.parts = 1;
    if (2 * p.real <= 148) {   // too few tiles: deal the key tiles to several CTAs, at least four each
        int64_t ns = 148 / p.real, most = keys / KT / 4;
        ns = ns < most ? ns : most;
        p.parts = (int)(ns > 32 ? 32 : (ns < 1 ? 1 : ns));
    }
    return p;
}

cudaError_t attn4_tc_launch(Attn4Args a, const b200seq_step& st, const Attn4TcPlan& p, cudaStream_t cs) {
    a.Rb = p.Rb, a.HB = p.HB, a.QT = p.QT, a.parts = p.parts;
    const dim3 grid((unsigned)(a.G * p.HB * p.tiles), 1, (unsigned)p.parts);
    const int nk = kv4_groups(a.D);
    if (p.mt == 2) return nk == 1 ? run<2, 1, 1>(a, st, grid, cs) : run<2, 2, 2>(a, st, grid, cs);
    return nk == 1 ? run<1, 1, 1>(a, st, grid, cs) : (nk == 2 ? run<1, 2, 2>(a, st, grid, cs) : run<1, 4, 4>(a, st, grid, cs));
}

}  // namespace b200seq
