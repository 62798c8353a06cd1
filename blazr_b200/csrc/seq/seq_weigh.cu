// seq_weigh.cu -- the soft-max weight that a step's tokens give to every cached key of their sequence, added up per key head (what eviction goes by).
//
// acc[slot][g][j] += sum over the entry's tokens t (all, or its last few) and the query heads h of key head g of  p_thj = exp(z_thj) / (sum_j' exp(z_thj') + exp(sink_h)),
// z = softcap(scale * head_scale_h * q_th . k_j) over the keys that t sees; a key that the step itself brought gets the sum instead of having it added.
//
// Few rows a key head (rows path): bound by the keys' bytes.  A block has 128 keys, a warp 16 of them in registers (8 lanes to a key, so that a product of a row with 16 keys
// needs four shuffles), and goes through the rows, which lie in shared memory in the lanes' order; f32 multiply-adds.  It leaves 2^(z - its maximum), the maximum and the sum for
// every row in the work area; a second launch has every row's denominator from the blocks' and adds the weights up, key by key, the rows in their order: no atomics.  The work
// area's traffic is a row's 4 bytes a key against the key's 4 D bytes.
// Many rows: seq_weigh_tc.cu.  What neither takes (heads above 128 or of odd sizes) goes through f32 tiles here, twice: once for the denominators, once for the sums.
#include "seq_weigh.cuh"
#include "tc_split.cuh"

namespace b200seq {

namespace {

using tcsplit::ex2;

// ---- rows path ------------------------------------------------------------------------------------------------------------------------------
constexpr int RT = 256;                // threads
constexpr int RK = 128;                // keys of a block
constexpr int RROWS = 32;              // rows in shared memory at a time
constexpr int FT = 256, FK = 4 * FT;   // second launch: threads, keys of a block

// work area of the rows path: [T][H][blocks][RK] weights relative to the block's maximum, then [T][H][blocks] (maximum, sum)
__device__ __forceinline__ float* rows_weights(const WeighArgs& a, int64_t row) { return a.part + row * a.key_blocks * RK; }
__device__ __forceinline__ float2* rows_stats(const WeighArgs& a, int T, int64_t row) {
    return reinterpret_cast<float2*>(a.part + (int64_t)T * a.H * a.key_blocks * RK) + row * a.key_blocks;
}

// grid (blocks of keys, key heads, entries).  VPL: values of a key in a lane (8 lanes to a key); FOUR: 4-bit pages
template <int VPL, bool FOUR>
__global__ void __launch_bounds__(RT, 2) weigh_rows_kernel(const __grid_constant__ WeighArgs a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    constexpr int Q = VPL / 4;          // 16-byte pieces of a lane
    __shared__ __align__(16) float qs[RROWS][VPL * 8];
    __shared__ float zs[RROWS][RK];
    __shared__ float factor[RROWS];
    const int e = blockIdx.z, g = blockIdx.y, k0 = blockIdx.x * RK, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const WeighEntry en(a, st, e, blockIdx.x == 0 && g == 0 && tid == 0);
    if (en.n == 0 || k0 >= en.keys) return;
    const int R = a.H / a.G, rows = en.n * R, bs = st.block_size, l8 = lane & 7, hi = en.keys - 1;
    const int32_t* bt = st.block_table + (int64_t)e * st.max_blocks;
    float k[4][VPL];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int key = min(k0 + warp * 16 + j * 4 + (lane >> 3), hi), page = kv4_page_read(bt[key / bs], a.err), o = key % bs;
        if (FOUR) {
            const Kv4Row r = kv4_row(page, o, bs, g, a.G, a.NG);
            constexpr int W = VPL / 8;  // words of a lane; a row has 4 NG of them, so that lanes behind NG / W * 4 have none
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int word = l8 * W + w, grp = word % a.NG;
                uint32_t c = 0, par = 0;
                if (word < 4 * a.NG) {
                    c = *reinterpret_cast<const uint32_t*>(a.kpool4 + r.codes + 4 * word);
                    par = *reinterpret_cast<const uint32_t*>(a.kpool4 + r.params + 4 * grp);
                }
                const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&par));
#pragma unroll
                for (int i = 0; i < 8; ++i) k[j][w * 8 + i] = fmaf((float)((c >> (4 * i)) & 15u), sm.x, sm.y);
            }
        } else {
            const float* row = a.kpool + (((int64_t)page * bs + o) * a.G + g) * a.D;
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const int d = (i * 8 + l8) * 4;
                const float4 x = d < a.D ? ld4(row + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                k[j][4 * i] = x.x, k[j][4 * i + 1] = x.y, k[j][4 * i + 2] = x.z, k[j][4 * i + 3] = x.w;
            }
        }
    }
    for (int r0 = 0; r0 < rows; r0 += RROWS) {
        const int nr = min(RROWS, rows - r0);
        __syncthreads();
        // queries in the lanes' order: piece i of lane l at [(i * 8 + l) * 4]
        for (int i = tid; i < nr * VPL * 8; i += RT) {
            const int r = i / (VPL * 8), s = i - r * (VPL * 8), x = s & 3, piece = s >> 2, l = piece & 7, pc = piece >> 3;
            int d;
            if (FOUR) {
                const int v = pc * 4 + x, word = l * (VPL / 8) + v / 8;
                d = word < 4 * a.NG ? 32 * (word % a.NG) + 8 * (word / a.NG) + v % 8 : a.D;
            } else {
                d = piece * 4 + x;
            }
            const int row = r0 + r, t = en.t0 + row / R, h = g * R + row % R;
            qs[r][s] = d < a.D ? a.q[(int64_t)t * a.ld + (int64_t)h * a.D + d] : 0.f;
        }
        if (tid < nr) factor[tid] = weigh_factor(a, g * R + (r0 + tid) % R);
        __syncthreads();
#pragma unroll 1
        for (int r = 0; r < nr; ++r) {
            uint64_t s[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                const float4 x = ld4(&qs[r][(i * 8 + l8) * 4]);
                const uint64_t x0 = tcsplit::pk(x.x, x.y), x1 = tcsplit::pk(x.z, x.w);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    s[j] = tcsplit::fma2(tcsplit::pk(k[j][4 * i], k[j][4 * i + 1]), x0, s[j]), s[j] = tcsplit::fma2(tcsplit::pk(k[j][4 * i + 2], k[j][4 * i + 3]), x1, s[j]);
            }
            float p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float u, v;
                tcsplit::upk(s[j], u, v);
                p[j] = u + v;
            }
            // four sums over eight lanes: lanes with bits (b2, b1) end up with key 2 b2 + b1's
            const bool b2 = lane & 4, b1 = lane & 2;
            float v0 = (b2 ? p[2] : p[0]) + __shfl_xor_sync(0xffffffffu, b2 ? p[0] : p[2], 4);
            float v1 = (b2 ? p[3] : p[1]) + __shfl_xor_sync(0xffffffffu, b2 ? p[1] : p[3], 4);
            float w = (b1 ? v1 : v0) + __shfl_xor_sync(0xffffffffu, b1 ? v0 : v1, 2);
            w += __shfl_xor_sync(0xffffffffu, w, 1);
            if (!(lane & 1)) zs[r][warp * 16 + ((lane >> 1) & 3) * 4 + (lane >> 3)] = weigh_score(w, factor[r], a.softcap);
        }
        __syncthreads();
        for (int r = warp; r < nr; r += RT / 32) {
            const int row = r0 + r, t = en.t0 + row / R, h = g * R + row % R;
            const WeighSpan span(a, en.p0 + row / R);
            float z[4], m = -INFINITY, l = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                z[i] = zs[r][4 * lane + i];
                if (!span.sees(k0 + 4 * lane + i)) z[i] = -INFINITY;
                m = fmaxf(m, z[i]);
            }
            m = warp_max(m);
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = z[i] == -INFINITY ? 0.f : ex2(z[i] - m), l += z[i];
            l = warp_sum(l);
            const int64_t at = (int64_t)t * a.H + h;
            *reinterpret_cast<float4*>(rows_weights(a, at) + k0 + 4 * lane) = make_float4(z[0], z[1], z[2], z[3]);
            if (lane == 0) rows_stats(a, st.T, at)[blockIdx.x] = make_float2(m, l);
        }
    }
}

// grid (blocks of FK keys, key heads, entries)
__global__ void __launch_bounds__(FT) weigh_join_kernel(const __grid_constant__ WeighArgs a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    constexpr int PER = FK / RK;
    __shared__ float f[RROWS][PER];
    const int e = blockIdx.z, g = blockIdx.y, k0 = blockIdx.x * FK, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const WeighEntry en(a, st, e, false);
    if (en.n == 0 || k0 >= en.keys) return;
    const int R = a.H / a.G, rows = en.n * R, nb = (en.keys + RK - 1) / RK, b0 = blockIdx.x * PER;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const int key = k0 + 4 * tid;
    for (int r0 = 0; r0 < rows; r0 += RROWS) {
        const int nr = min(RROWS, rows - r0);
        __syncthreads();
        for (int r = warp; r < nr; r += FT / 32) {      // factors of the blocks' weights: 2^(the block's maximum - lse)
            const int row = r0 + r, h = g * R + row % R;
            const float2* s = rows_stats(a, st.T, (int64_t)(en.t0 + row / R) * a.H + h);
            float m = -INFINITY, l = 0.f;
            for (int i = lane; i < nb; i += 32) m = fmaxf(m, s[i].x);
            m = warp_max(m);
            for (int i = lane; i < nb; i += 32) {
                const float2 x = s[i];
                l += x.x == -INFINITY ? x.y : x.y * ex2(x.x - m);      // (a block without a key to see: 0, or no number)
            }
            l = warp_sum(l);
            float den = l, top = m;
            if (a.sink) {
                const float sk = a.sink[h] * WEIGH_LOG2E;
                top = fmaxf(m, sk);
                den = (m == -INFINITY ? l : l * ex2(m - top)) + ex2(sk - top);
            }
            if (lane < PER && b0 + lane < nb) {
                const float bm = s[b0 + lane].x;
                f[r][lane] = bm == -INFINITY ? (l == l ? 0.f : l) : ex2(bm - top) / den;
            }
        }
        __syncthreads();
        if (key < en.keys) {
#pragma unroll 4
            for (int r = 0; r < nr; ++r) {
                const int row = r0 + r;
                const float4 w = ld4(rows_weights(a, (int64_t)(en.t0 + row / R) * a.H + g * R + row % R) + key);
                const float x = f[r][4 * tid / RK];
                sum.x = fmaf(w.x, x, sum.x), sum.y = fmaf(w.y, x, sum.y), sum.z = fmaf(w.z, x, sum.z), sum.w = fmaf(w.w, x, sum.w);
            }
        }
    }
    float* acc = a.acc + ((int64_t)en.slot * a.G + g) * a.acc_ld;
    const float s[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (key + i < en.keys) acc[key + i] = key + i < en.fresh ? acc[key + i] + s[i] : s[i];
}

// ---- f32 tiles ------------------------------------------------------------------------------------------------------------------------------
constexpr int TT = 256, TK = 64, TR = 32, SLAB = 32;      // threads, keys and rows of a tile, values of a slab

struct Tile {
    float k[TK][SLAB + 1], q[TR][SLAB + 1];
};

__device__ __forceinline__ float key_value_at(const WeighArgs& a, int page, int o, int bs, int g, int d, bool four) {
    if (!four) return a.kpool[(((int64_t)page * bs + o) * a.G + g) * a.D + d];
    const Kv4Row r = kv4_row(page, o, bs, g, a.G, a.NG);
    const int word = (d % 32 / 8) * a.NG + d / 32;
    const uint32_t c = *reinterpret_cast<const uint32_t*>(a.kpool4 + r.codes + 4 * word), par = *reinterpret_cast<const uint32_t*>(a.kpool4 + r.params + 4 * (d / 32));
    const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&par));
    return fmaf((float)((c >> (4 * (d % 8))) & 15u), sm.x, sm.y);
}

// dot products of a tile: keys tid % 16 + 16 i, rows 2 (tid / 16) + r in dot[i][r]
__device__ __forceinline__ void tile_dots(const WeighArgs& a, const b200seq_step& st, const WeighEntry& en, int e, int g, int k0, int row0, bool four, Tile& t, float (&dot)[4][2]) {
    const int tid = threadIdx.x, R = a.H / a.G, rows = en.n * R, bs = st.block_size;
    const int32_t* bt = st.block_table + (int64_t)e * st.max_blocks;
#pragma unroll
    for (int i = 0; i < 4; ++i) dot[i][0] = dot[i][1] = 0.f;
    for (int d0 = 0; d0 < a.D; d0 += SLAB) {
        __syncthreads();
        for (int i = tid; i < TK * SLAB; i += TT) {
            const int key = min(k0 + i / SLAB, en.keys - 1), d = d0 + i % SLAB;
            t.k[i / SLAB][i % SLAB] = d < a.D ? key_value_at(a, kv4_page_read(bt[key / bs], a.err), key % bs, bs, g, d, four) : 0.f;
        }
        for (int i = tid; i < TR * SLAB; i += TT) {
            const int row = row0 + i / SLAB, d = d0 + i % SLAB;
            t.q[i / SLAB][i % SLAB] = row < rows && d < a.D ? a.q[(int64_t)(en.t0 + row / R) * a.ld + (int64_t)(g * R + row % R) * a.D + d] : 0.f;
        }
        __syncthreads();
#pragma unroll 8
        for (int d = 0; d < SLAB; ++d) {
            const float q0 = t.q[2 * (tid >> 4)][d], q1 = t.q[2 * (tid >> 4) + 1][d];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float k = t.k[(tid & 15) + 16 * i][d];
                dot[i][0] = fmaf(k, q0, dot[i][0]), dot[i][1] = fmaf(k, q1, dot[i][1]);
            }
        }
    }
}

// grid (row tiles of the longest entry, key heads, entries): denominators
__global__ void __launch_bounds__(TT) weigh_tile_lse_kernel(const __grid_constant__ WeighArgs a, const __grid_constant__ b200seq_step st, int four) {
    chain_enter();
    __shared__ Tile tile;
    const int e = blockIdx.z, g = blockIdx.y, row0 = blockIdx.x * TR, tid = threadIdx.x;
    const WeighEntry en(a, st, e, blockIdx.x == 0 && g == 0 && tid == 0);
    const int R = a.H / a.G, rows = en.n * R;
    if (row0 >= rows) return;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int pmax = en.p0 + min(rows - 1, row0 + TR - 1) / R;
    for (int k0 = 0; k0 <= pmax; k0 += TK) {
        const WeighSpan first(a, en.p0 + row0 / R);
        if (k0 + TK <= first.lo && k0 >= first.keep) continue;         // no row of the tile sees these keys
        float dot[4][2];
        tile_dots(a, st, en, e, g, k0, row0, four, tile, dot);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = row0 + 2 * (tid >> 4) + r;
            if (row >= rows) continue;
            const WeighSpan span(a, en.p0 + row / R);
            const float fac = weigh_factor(a, g * R + row % R);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!span.sees(k0 + (tid & 15) + 16 * i)) continue;
                const float z = weigh_score(dot[i][r], fac, a.softcap);
                if (z > m[r]) l[r] = m[r] == -INFINITY ? l[r] : l[r] * ex2(m[r] - z), m[r] = z;
                if (z != -INFINITY) l[r] += ex2(z - m[r]);
            }
        }
    }
    // sixteen neighbouring lanes share a pair of rows
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = row0 + 2 * (tid >> 4) + r;
        float top = m[r];
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float s = m[r] == -INFINITY ? l[r] : l[r] * ex2(m[r] - top);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if ((tid & 15) == 0 && row < rows) {
            const int h = g * R + row % R;
            a.lse[(int64_t)(en.t0 + row / R) * a.H + h] = s != s ? s : weigh_lse(a, h, top, s);
        }
    }
}

// grid (key tiles of the longest sequence, key heads, entries): sums
__global__ void __launch_bounds__(TT) weigh_tile_sum_kernel(const __grid_constant__ WeighArgs a, const __grid_constant__ b200seq_step st, int four) {
    chain_enter();
    __shared__ Tile tile;
    __shared__ float part[TT / 16][TK];
    const int e = blockIdx.z, g = blockIdx.y, k0 = blockIdx.x * TK, tid = threadIdx.x;
    const WeighEntry en(a, st, e, false);
    if (en.n == 0 || k0 >= en.keys) return;
    const int R = a.H / a.G, rows = en.n * R;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int row0 = 0; row0 < rows; row0 += TR) {
        const int p1 = en.p0 + min(rows - 1, row0 + TR - 1) / R;
        const WeighSpan first(a, en.p0 + row0 / R);
        if (p1 < k0 || (k0 + TK <= first.lo && k0 >= first.keep)) continue;
        float dot[4][2];
        tile_dots(a, st, en, e, g, k0, row0, four, tile, dot);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = row0 + 2 * (tid >> 4) + r;
            if (row >= rows) continue;
            const int h = g * R + row % R;
            const WeighSpan span(a, en.p0 + row / R);
            const float fac = weigh_factor(a, h), lse = a.lse[(int64_t)(en.t0 + row / R) * a.H + h];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (span.sees(k0 + (tid & 15) + 16 * i) && lse != -INFINITY) sum[i] += ex2(weigh_score(dot[i][r], fac, a.softcap) - lse);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) part[tid >> 4][(tid & 15) + 16 * i] = sum[i];
    __syncthreads();
    if (tid < TK && k0 + tid < en.keys) {
        float s = 0.f;
        for (int i = 0; i < TT / 16; ++i) s += part[i][tid];
        float* acc = a.acc + ((int64_t)en.slot * a.G + g) * a.acc_ld + k0 + tid;
        *acc = k0 + tid < en.fresh ? *acc + s : s;
    }
}

int check(const b200seq_step* st, const b200seq_attn_desc* d, int kv_bits) {
    if (!st || st->T < 0 || st->B < 0 || st->max_blocks < 1 || st->block_size < 1) return fail(B200SEQ_ERR_INVALID_ARG, "key_weights: bad step");
    if (int rc = attn_desc_check(d, "key_weights")) return rc;
    if (kv_bits != 4 && kv_bits != 32) return fail(B200SEQ_ERR_INVALID_ARG, "key_weights: a cache of 4 or 32 bits a value, not %d", kv_bits);
    if (d->pool > 0 || d->latent_v || d->ctx_rows || d->krot || (d->kv_ld > 0 && d->kv_ld != (int64_t)d->G * d->D))
        return fail(B200SEQ_ERR_UNSUPPORTED, "key_weights: plain keys in pages, not pooled blocks, latents or gathered rows");
    if (kv_bits == 4 && (d->D > KV4_MAX_DIM || !kv4_pages_fit(st->block_size, d->G, d->D))) return fail(B200SEQ_ERR_UNSUPPORTED, "key_weights: 4-bit pages hold heads of up to %d values", KV4_MAX_DIM);
    if (st->B > 65535 || d->G > 65535) return fail(B200SEQ_ERR_UNSUPPORTED, "key_weights: up to 65535 entries and key heads");
    return 0;
}

// How a step is run.  Rows that share a key head in one entry: up to ROWS_MOST go through the rows path, whose time grows with them, if its weights fit the work area that it may have.
constexpr int ROWS_MOST = 64;
constexpr int64_t ROWS_FLOATS = 64 << 20;
struct Plan {
    bool rows;
    int blocks;        // rows path: blocks of RK keys of the longest sequence
    int tokens;        // tokens of an entry that count: a bound
    WeighTcPlan tc;
    size_t floats;
};
Plan plan_of(const b200seq_step& st, const b200seq_attn_desc& d, int last, int max_keys) {
    Plan p;
    const int64_t held = (int64_t)st.max_blocks * st.block_size;
    const int64_t keys = max_keys > 0 && max_keys < held ? max_keys : held;
    p.blocks = (int)((keys + RK - 1) / RK);
    const int each = (st.T + st.B - 1) / (st.B > 0 ? st.B : 1), tokens = last > 0 && last < each ? last : each;      // (were all entries equally long)
    p.tokens = last > 0 && last < st.T ? last : st.T;
    const int64_t floats = (int64_t)st.T * d.H * p.blocks * (RK + 2);
    p.rows = d.D <= 128 && (int64_t)tokens * (d.H / d.G) <= ROWS_MOST && floats <= ROWS_FLOATS;
    p.tc = weigh_tc_plan(st, d.H, d.G, last, (int64_t)p.blocks * RK);
    p.floats = p.rows ? (size_t)floats : p.tc.floats;      // (more than the f32 tiles' T * H)
    return p;
}

}  // namespace

}  // namespace b200seq

using namespace b200seq;

extern "C" {

size_t b200seq_key_weights_scratch_floats(const b200seq_step* st, const b200seq_attn_desc* d, int last, int max_keys) {
    if (!st || !d || st->T < 1 || st->B < 1 || d->H < 1 || d->G < 1 || st->max_blocks < 1 || st->block_size < 1) return 0;
    return plan_of(*st, *d, last, max_keys).floats;
}

int b200seq_key_weights(const float* proj, int64_t ld, const b200seq_step* st, const b200seq_attn_desc* d, const void* kpool, int kv_bits, float* acc, int slots, int64_t acc_ld,
                        int last, int max_keys, float* scratch, size_t scratch_floats, void* stream) {
    if (int rc = check(st, d, kv_bits)) return rc;
    if (!proj || !kpool || !acc || slots < 1 || acc_ld < 1 || last < 0 || max_keys < 0) return fail(B200SEQ_ERR_INVALID_ARG, "key_weights: bad arguments");
    if (st->T == 0 || st->B == 0) return 0;
    if (ld < (int64_t)d->q_col + (int64_t)d->H * d->D && st->T > 1) return fail(B200SEQ_ERR_INVALID_ARG, "key_weights: row stride below the queries' columns");
    const Plan p = plan_of(*st, *d, last, max_keys);
    if (!scratch || scratch_floats < p.floats || (reinterpret_cast<uintptr_t>(scratch) & 15)) return fail(B200SEQ_ERR_INVALID_ARG, "key_weights: the work area is too small or not on a 16-byte boundary");
    const bool four = kv_bits == 4;
    if (four && (reinterpret_cast<uintptr_t>(kpool) & 15)) return fail(B200SEQ_ERR_INVALID_ARG, "key_weights: 4-bit pools start on a 16-byte boundary");
    const cudaStream_t cs = (cudaStream_t)stream;
    WeighArgs a = {};
    a.q = proj + d->q_col, a.ld = ld, a.kpool = (const float*)kpool, a.kpool4 = (const uint8_t*)kpool, a.acc = acc, a.acc_ld = acc_ld, a.slots = slots;
    a.H = d->H, a.G = d->G, a.D = d->D, a.NG = four ? kv4_groups(d->D) : 0, a.last = last, a.scale = d->scale, a.softcap = d->softcap;
    a.chunk = d->chunk, a.window = d->window, a.keep_first = d->keep_first, a.head_scale = d->head_scale, a.sink = d->sink, a.most_keys = (int64_t)p.blocks * RK, a.err = error_flag_dev();
    const bool wide = four || ((d->D & 3) == 0 && (reinterpret_cast<uintptr_t>(kpool) & 15) == 0);
    if (p.rows && wide) {
        a.part = scratch, a.key_blocks = p.blocks;
        const dim3 grid(p.blocks, d->G, st->B);
        if (four) {
            if (d->D <= 64) launch_chained(weigh_rows_kernel<8, true>, grid, RT, 0, cs, a, *st);
            else launch_chained(weigh_rows_kernel<16, true>, grid, RT, 0, cs, a, *st);
        } else {
            if (d->D <= 64) launch_chained(weigh_rows_kernel<8, false>, grid, RT, 0, cs, a, *st);
            else launch_chained(weigh_rows_kernel<16, false>, grid, RT, 0, cs, a, *st);
        }
        SEQ_LAUNCH_CHECK("key_weights");
        launch_chained(weigh_join_kernel, dim3((p.blocks * RK + FK - 1) / FK, d->G, st->B), FT, 0, cs, a, *st);
        SEQ_LAUNCH_CHECK("key_weights");
        return 0;
    }
    if (weigh_tc_takes(a, four)) return weigh_tc(a, *st, p.tc, scratch, four, cs);
    a.lse = scratch;
    const int64_t tiles = ((int64_t)p.tokens * (d->H / d->G) + TR - 1) / TR, key_tiles = (p.blocks * (int64_t)RK + TK - 1) / TK;
    launch_chained(weigh_tile_lse_kernel, dim3((unsigned)tiles, d->G, st->B), TT, 0, cs, a, *st, (int)four);
    SEQ_LAUNCH_CHECK("key_weights");
    launch_chained(weigh_tile_sum_kernel, dim3((unsigned)key_tiles, d->G, st->B), TT, 0, cs, a, *st, (int)four);
    SEQ_LAUNCH_CHECK("key_weights");
    return 0;
}

}  // extern "C"
