// seq_weigh.cu -- the soft-max weight that a step's tokens give to every cached key of their sequence, added up per key head (what eviction goes by).
//
// acc[slot][g][j] += sum over the entry's tokens t (all, or its last few) and the query heads h of key head g of  p_thj = exp(z_thj) / (sum_j' exp(z_thj') + exp(sink_h)),
// z = softcap(scale * head_scale_h * q_th . k_j) over the keys that t sees; a key that the step itself brought gets the sum instead of having it added.
//
// Few rows a key head (rows path): bound by the keys' bytes.  Eight rows are too few for a tcgen05 product of 128: a warp takes eight keys at a time into registers, a lane a quarter of one,
// splits them there into two f16 parts (k = h + l, l times 2^11) and multiplies with m16n8k16 products, whose rows 0 - 7 are the high parts of eight rows of queries and 8 - 15 their
// low parts (times 2^11), so that two products a step give all four: 22 bits, at any size of the keys that f16 has.  What has no such parts gives no number and is made again in f32.  The scores
// go to the work area (4 bytes a row and key against the key's 4 D), with every block's maximum and sum a row; a second launch has every row's denominator from the blocks' and
// adds the weights up, key by key, the rows in their order: no atomics.
// Measured: 32 sequences of 2000 to 4000 keys, 32 query heads of 8 key heads of 128, 88 to 91 us (75 and 11, 5.4 TB/s of keys in the first), one of 131072 keys 116 to 121 (100
// and 15; 4.5 TB/s over both); what the first launch spends are instructions: 364 of a warp for eight keys, two a cycle and SM.  (In f32 multiply-adds: 123 and 149.)
// Many rows: seq_weigh_tc.cu.  What neither takes (heads above 128 or of odd sizes) goes through f32 tiles here, twice: once for the denominators, once for the sums.
#include <cooperative_groups.h>

#include "seq_weigh.cuh"
#include "tc_split.cuh"

namespace b200seq {

namespace {

using tcsplit::ex2;

// ---- rows path ------------------------------------------------------------------------------------------------------------------------------
constexpr int RT = 256, RW = RT / 32;  // threads, warps
constexpr int FT = 256, FK = 4 * FT;   // second launch: threads, keys of a block
constexpr int MOST_TILES = 16;         // of eight keys of a warp
constexpr float LOW = 0x1p11f, UNLOW = 0x1p-11f;

// the base-2 logarithm of a row's denominator from its maximum and sum; infinite where the row gives nothing
__device__ __forceinline__ float denominator(const WeighArgs& a, int h, float m, float l) {
    if (l != l) return l;
    const float v = weigh_lse(a, h, m, l);
    return v == -INFINITY ? INFINITY : v;
}

// work area of the rows path: [T][H][key_room] scores in base 2, then [T][H][key_blocks] (maximum, sum)
__device__ __forceinline__ float* rows_scores(const WeighArgs& a, int64_t row) { return a.part + row * a.key_room; }
__device__ __forceinline__ float2* rows_stats(const WeighArgs& a, int T, int64_t row) { return reinterpret_cast<float2*>(a.part + (int64_t)T * a.H * a.key_room) + row * a.key_blocks; }

__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// two values -> f16 pair of their high parts and f16 pair of what is left times 2^11 (low half = a)
__device__ __forceinline__ void split_up(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    float x, y;      // (x - h) 2^11: both products are exact
    tcsplit::upk(tcsplit::fma2(tcsplit::pk(f.x, f.y), tcsplit::pk(-LOW, -LOW), tcsplit::mul2(tcsplit::pk(a, b), tcsplit::pk(LOW, LOW))), x, y);
    const __half2 l = __floats2half2_rn(x, y);
    hi = *reinterpret_cast<const uint32_t*>(&h), lo = *reinterpret_cast<const uint32_t*>(&l);
}

// What a lane has of a key (c: lane & 3).  4-bit keys: of every group of 32 values the eight from 8 c on, codes and parameters in registers, a tile ahead.  f32 ones: of every 16 values the
// four from 4 c on, on their way to the lane's own places of a ring in shared memory, two tiles ahead (in registers there was room for one: with eight tiles a warp 32 sequences 97 us, now 93; one of 131072
// keys 119 either way).
constexpr int RING = 3;
template <int NG, bool FOUR>
struct KeyPart {
    uint32_t code[FOUR ? NG : 1], par[FOUR ? NG : 1];
    __device__ __forceinline__ void fetch(const WeighArgs& a, int page, int o, int bs, int g, int c) {
        const Kv4Row r = kv4_row(page, o, bs, g, a.G, NG);
        const uint8_t *k = a.kpool4 + r.codes + c * NG * 4, *p = a.kpool4 + r.params;
        if constexpr (NG == 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(k), v = *reinterpret_cast<const uint4*>(p);
            code[0] = u.x, code[1] = u.y, code[2] = u.z, code[3] = u.w, par[0] = v.x, par[1] = v.y, par[2] = v.z, par[3] = v.w;
        } else if constexpr (NG == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(k), v = *reinterpret_cast<const uint2*>(p);
            code[0] = u.x, code[1] = u.y, par[0] = v.x, par[1] = v.y;
        } else {
            code[0] = *reinterpret_cast<const uint32_t*>(k), par[0] = *reinterpret_cast<const uint32_t*>(p);
        }
    }
    // the four values of step kk (two steps a group)
    __device__ __forceinline__ float4 step(int kk) const {
        const uint32_t w = code[kk >> 1] >> (16 * (kk & 1)), p = par[kk >> 1];
        const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&p));
        // (a code in the mantissa of 2^23: that number more)
        auto val = [&](uint32_t u) { return fmaf(__uint_as_float(u | 0x4B000000u) - 8388608.f, sm.x, sm.y); };
        return make_float4(val(w & 15u), val((w >> 4) & 15u), val((w >> 8) & 15u), val((w >> 12) & 15u));
    }
};
// pieces of an f32 key to `dst` + 512 i (places behind the head's values: zeros)
template <int NG>
__device__ __forceinline__ void fetch_key(const WeighArgs& a, uint32_t dst, int page, int o, int bs, int g, int c) {
    const float* row = a.kpool + (((int64_t)page * bs + o) * a.G + g) * a.D + 4 * c;
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i) {
        const int d = 16 * i;
        const bool in = d + 4 * c < a.D;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 512 * i), "l"(in ? row + d : a.kpool), "r"(in ? 16 : 0) : "memory");
    }
}

// grid (blocks of 64 * tiles keys, key heads, entries).  NRT: tiles of eight rows that are gone through at a time.  JOINED: a sequence's blocks are one cluster, which joins their
// maxima and sums itself and adds the weights up at once.  (For steps whose blocks are all on the GPU together, two an SM: one token of 500 keys 14.2 -> 11.7 us; in several waves the
// blocks that wait for one another keep others out, 32 sequences 88 -> 137.  With four tiles of rows and f32 keys of more than 64 values a block has 117 KB of shared memory and
// an SM one block; joined steps are then the faster ones up to two waves.  Waves of clusters leave SMs idle: 30 clusters of eight, 40 of six, 64 of four and 144 of two take 22 us for
// 25 to 26 in two launches, 32, 48 and 72 of the first three 31, 57 for 46 (64 rows) and 31.)
template <int NRT, int NG, bool FOUR, bool JOINED>
__global__ void __launch_bounds__(RT, 2) weigh_rows_kernel(const __grid_constant__ WeighArgs a, const __grid_constant__ b200seq_step st, int tiles) {
    chain_enter();
    extern __shared__ __align__(16) float4 ring[];      // f32: [warp][RING][2 NG][lane]
    __shared__ uint4 frag[NRT][2 * NG][32];
    __shared__ float2 part[RW][NRT * 8], fin[NRT * 8];
    __shared__ float den[NRT * 8];
    const int e = blockIdx.z, g = blockIdx.y, k0 = blockIdx.x * 64 * tiles, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = lane & 3, r8 = lane >> 2;
    const WeighEntry en(a, st, e, blockIdx.x == 0 && g == 0 && tid == 0);
    if (en.n == 0 || (k0 >= en.keys && !JOINED)) return;      // (a cluster's blocks stay together)
    const int R = a.H / a.G, rows = en.n * R, bs = st.block_size, hi = en.keys - 1;
    float total[MOST_TILES / 4];                             // JOINED: the weights of keys k0 + tid + 256 q
#pragma unroll
    for (int q = 0; q < MOST_TILES / 4; ++q) total[q] = 0.f;
    const int32_t* bt = st.block_table + (int64_t)e * st.max_blocks;
    // a warp's keys: k0 + 8 (warp + 8 i) ..., of which a lane has key lane / 4
    // (place in the table and row of the page of the next one that is looked up, and of the next one that is fetched: 64 keys on each time, without a division)
    const int key_first = k0 + 8 * warp + r8, on_pages = 64 / bs, on_rows = 64 - on_pages * bs, hi_page = hi / bs, hi_row = hi - hi_page * bs;
    int look_page, look_row, row_page, row_row;
    auto restart = [&]() { look_page = row_page = key_first / bs, look_row = row_row = key_first - look_page * bs; };
    auto next_page = [&]() {      // pages in the order of the tiles (behind the last key: its page)
        const int page = kv4_page_read(bt[min(look_page, hi_page)], a.err);
        look_page += on_pages, look_row += on_rows;
        if (look_row >= bs) look_row -= bs, ++look_page;
        return page;
    };
    auto next_row = [&]() {       // and rows
        const int row = row_page > hi_page || (row_page == hi_page && row_row > hi_row) ? hi_row : row_row;
        row_page += on_pages, row_row += on_rows;
        if (row_row >= bs) row_row -= bs, ++row_page;
        return row;
    };
    const bool cap = a.softcap > 0.f;
    for (int r0 = 0; r0 < rows; r0 += NRT * 8) {
        restart();
        KeyPart<NG, FOUR> nxt, cur;
        const float4* const mine = ring + warp * (RING * 2 * NG * 32) + lane;
        const uint32_t mine_at = tcpair::sa(mine);
        int page;
        if constexpr (FOUR) {
            page = next_page();
            nxt.fetch(a, page, next_row(), bs, g, c);
            page = tiles > 1 ? next_page() : 0;
        } else {
            const int first = next_page(), second = tiles > 1 ? next_page() : 0;
            page = tiles > 2 ? next_page() : 0;
            fetch_key<NG>(a, mine_at, first, next_row(), bs, g, c);
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (tiles > 1) fetch_key<NG>(a, mine_at + 1024 * NG, second, next_row(), bs, g, c);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        __syncthreads();
        for (int i = tid; i < NRT * 2 * NG * 32; i += RT) {
            const int ln = i & 31, kk = (i >> 5) % (2 * NG), rt = i / (64 * NG), row = r0 + 8 * rt + (ln >> 2);
            const int d = FOUR ? 32 * (kk >> 1) + 8 * (ln & 3) + 4 * (kk & 1) : 16 * kk + 4 * (ln & 3);
            uint4 f = make_uint4(0, 0, 0, 0);
            if (row < rows) {
                const int h = g * R + row % R;
                const float* q = a.q + (int64_t)(en.t0 + row / R) * a.ld + (int64_t)h * a.D;
                const float fac = weigh_factor(a, h) * (cap ? 1.f : WEIGH_LOG2E);
                float x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = d + j < a.D ? q[d + j] * fac : 0.f;
                split_up(x[0], x[1], f.x, f.y), split_up(x[2], x[3], f.z, f.w);
            }
            frag[rt][kk][ln] = f;
        }
        __syncthreads();
        float m[NRT], l[NRT];
        int pos[NRT], lo[NRT];
        float* out[NRT];
#pragma unroll
        for (int rt = 0; rt < NRT; ++rt) {
            const int row = r0 + 8 * rt + r8;
            const bool live = row < rows;
            const WeighSpan span(a, en.p0 + (live ? row / R : 0));
            m[rt] = -INFINITY, l[rt] = 0.f, pos[rt] = live ? span.p : -1, lo[rt] = span.lo;
            out[rt] = rows_scores(a, live ? (int64_t)(en.t0 + row / R) * a.H + g * R + row % R : 0);
        }
        const int keep = a.window > 0 ? a.keep_first : 0, pos_least = en.p0 + r0 / R;
        const WeighSpan last(a, en.p0 + min(rows - 1, r0 + NRT * 8 - 1) / R);
        const int lo_most = last.lo;
        int slot = 0;
#pragma unroll 1
        for (int i = 0; i < tiles; ++i) {
            const int key0 = k0 + 8 * (warp + RW * i);
            if (key0 > hi) break;
            const float4* const now = mine + slot * (2 * NG * 32);
            if constexpr (FOUR) {
                cur = nxt;
                if (i + 1 < tiles) {
                    nxt.fetch(a, page, next_row(), bs, g, c);
                    if (i + 2 < tiles) page = next_page();
                }
            } else {
                if (i + 2 < tiles) {
                    fetch_key<NG>(a, mine_at + (slot == 0 ? 2 : slot - 1) * (1024 * NG), page, next_row(), bs, g, c);
                    if (i + 3 < tiles) page = next_page();
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group 2;" ::: "memory");
                slot = slot == 2 ? 0 : slot + 1;
            }
            float ah[NRT][4], al[NRT][4];
#pragma unroll
            for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
                for (int j = 0; j < 4; ++j) ah[rt][j] = al[rt][j] = 0.f;
#pragma unroll
            for (int kk = 0; kk < 2 * NG; ++kk) {
                float4 x;
                if constexpr (FOUR) x = cur.step(kk);
                else x = now[kk * 32];
                uint32_t h0, h1, l0, l1;
                split_up(x.x, x.y, h0, l0), split_up(x.z, x.w, h1, l1);
#pragma unroll
                for (int rt = 0; rt < NRT; ++rt) {
                    const uint4 f = frag[rt][kk][lane];
                    mma16816(al[rt], f, l0, l1), mma16816(ah[rt], f, h0, h1);
                }
            }
            const int key = key0 + 2 * c;
            const bool whole = key0 >= lo_most && key0 + 7 <= pos_least;      // (every row sees all of the tile)
#pragma unroll
            for (int rt = 0; rt < NRT; ++rt) {
                float z[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    z[j] = fmaf(fmaf(al[rt][2 + j], UNLOW, al[rt][j] + ah[rt][2 + j]), UNLOW, ah[rt][j]);
                    if (cap) z[j] = a.softcap * WEIGH_LOG2E * tanhf(z[j] / a.softcap);
                }
                const bool odd = !(fabsf(z[0]) + fabsf(z[1]) < INFINITY);
                if (!whole || odd) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const bool sees = key + j <= pos[rt] && (key + j >= lo[rt] || key + j < keep);
                        if (!sees) z[j] = -INFINITY;
                        else if (odd) z[j] = plain_score(a, st, en, e, g, r0 + 8 * rt + r8, key + j, FOUR);
                    }
                }
                const float top = fmaxf(m[rt], fmaxf(z[0], z[1]));
                if (top > m[rt]) l[rt] *= ex2(m[rt] - top), m[rt] = top;
                const float off = m[rt] == -INFINITY ? 0.f : m[rt];      // (minus infinities give nothing)
                l[rt] += ex2(z[0] - off) + ex2(z[1] - off);
                if (pos[rt] >= 0) *reinterpret_cast<float2*>(out[rt] + key) = make_float2(z[0], z[1]);
            }
        }
        // (a warp that ran out of keys has copies on their way, to places that the next rows' copies go to as well: two copies to one place have no order)
        if constexpr (!FOUR) asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
        for (int rt = 0; rt < NRT; ++rt) {      // a row's four lanes, then the warps
            float top = m[rt];
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1)), top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            float s = m[rt] == -INFINITY ? l[rt] : l[rt] * ex2(m[rt] - top);
            s += __shfl_xor_sync(0xffffffffu, s, 1), s += __shfl_xor_sync(0xffffffffu, s, 2);
            if (c == 0) part[warp][8 * rt + r8] = make_float2(top, s);
        }
        __syncthreads();
        if (tid < NRT * 8 && r0 + tid < rows) {
            const int row = r0 + tid;
            float top = -INFINITY, s = 0.f;
            for (int w = 0; w < RW; ++w) top = fmaxf(top, part[w][tid].x);
            for (int w = 0; w < RW; ++w) {
                const float2 x = part[w][tid];
                s += x.x == -INFINITY ? x.y : x.y * ex2(x.x - top);
            }
            if constexpr (JOINED) fin[tid] = make_float2(top, s);
            else rows_stats(a, st.T, (int64_t)(en.t0 + row / R) * a.H + g * R + row % R)[blockIdx.x] = make_float2(top, s);
        }
        if constexpr (JOINED) {
            auto cl = cooperative_groups::this_cluster();
            cl.sync();                                      // (and this block's scores are written)
            if (tid < NRT * 8 && r0 + tid < rows) {
                float2 x[8];
                float top = -INFINITY, s = 0.f;
#pragma unroll
                for (int b = 0; b < 8; ++b) {
                    x[b] = b < (int)gridDim.x ? *cl.map_shared_rank(fin + tid, b) : make_float2(-INFINITY, 0.f);
                    top = fmaxf(top, x[b].x);
                }
#pragma unroll
                for (int b = 0; b < 8; ++b) s += x[b].x == -INFINITY ? x[b].y : x[b].y * ex2(x[b].x - top);
                den[tid] = denominator(a, g * R + (r0 + tid) % R, top, s);
            }
            __syncthreads();
            const int nr = min(NRT * 8, rows - r0);
#pragma unroll
            for (int q = 0; q < MOST_TILES / 4; ++q) {
                const int at = tid + RT * q, key = k0 + at;
                if (at >= 64 * tiles || key > hi) continue;
#pragma unroll 8
                for (int r = 0; r < nr; ++r) total[q] += ex2(rows_scores(a, (int64_t)(en.t0 + (r0 + r) / R) * a.H + g * R + (r0 + r) % R)[key] - den[r]);
            }
            cl.sync();                                      // nobody's sums go while they are read
        }
    }
    if constexpr (JOINED) {
        float* acc = a.acc + ((int64_t)en.slot * a.G + g) * a.acc_ld;
#pragma unroll
        for (int q = 0; q < MOST_TILES / 4; ++q) {
            const int at = tid + RT * q, key = k0 + at;
            if (at < 64 * tiles && key <= hi) acc[key] = key < en.fresh ? acc[key] + total[q] : total[q];
        }
    }
}

// grid (blocks of FK keys, key heads, entries)
__global__ void __launch_bounds__(FT, 3) weigh_join_kernel(const __grid_constant__ WeighArgs a, const __grid_constant__ b200seq_step st, int block_keys) {
    chain_enter();
    constexpr int ROWS = 32;
    __shared__ float den[ROWS];
    const int e = blockIdx.z, g = blockIdx.y, k0 = blockIdx.x * FK, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const WeighEntry en(a, st, e, false);
    if (en.n == 0 || k0 >= en.keys) return;
    const int R = a.H / a.G, rows = en.n * R, nb = (en.keys + block_keys - 1) / block_keys;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const int key = k0 + 4 * tid;
    auto score = [&](int row) { return ld4(rows_scores(a, (int64_t)(en.t0 + row / R) * a.H + g * R + row % R) + key); };
    // (the first rows' scores and the weights so far are on their way while the denominators are made)
    constexpr int AHEAD = 8;
    float* acc = a.acc + ((int64_t)en.slot * a.G + g) * a.acc_ld;
    float4 ahead[AHEAD];
    float old[4];
#pragma unroll
    for (int r = 0; r < AHEAD; ++r)
        if (key < en.keys && r < rows) ahead[r] = score(r);
#pragma unroll
    for (int i = 0; i < 4; ++i) old[i] = key + i < en.fresh ? acc[key + i] : 0.f;
    for (int r0 = 0; r0 < rows; r0 += ROWS) {
        const int nr = min(ROWS, rows - r0);
        __syncthreads();
        for (int r = warp; r < nr; r += FT / 32) {      // the rows' denominators (base-2 logarithms)
            const int row = r0 + r, h = g * R + row % R;
            const float2* s = rows_stats(a, st.T, (int64_t)(en.t0 + row / R) * a.H + h);
            float m = -INFINITY, l = 0.f;
#pragma unroll 8
            for (int i = lane; i < nb; i += 32) m = fmaxf(m, s[i].x);
            const float top = warp_max(m);
#pragma unroll 8
            for (int i = lane; i < nb; i += 32) {
                const float2 x = s[i];
                l += x.x == -INFINITY ? x.y : x.y * ex2(x.x - top);      // (a block without a key to see: 0, or no number)
            }
            l = warp_sum(l);
            if (lane == 0) den[r] = denominator(a, h, top, l);
        }
        __syncthreads();
        if (key < en.keys) {
            auto add = [&](const float4& z, float x) { sum.x += ex2(z.x - x), sum.y += ex2(z.y - x), sum.z += ex2(z.z - x), sum.w += ex2(z.w - x); };
            if (r0 == 0) {
#pragma unroll
                for (int r = 0; r < AHEAD; ++r)
                    if (r < nr) add(ahead[r], den[r]);
            }
#pragma unroll 4
            for (int r = r0 == 0 ? AHEAD : 0; r < nr; ++r) add(score(r0 + r), den[r]);
        }
    }
    const float s[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (key + i < en.keys) acc[key + i] = old[i] + s[i];
}

// How a step is run.  Rows that share a key head in one entry: up to ROWS_MOST go through the rows path, whose time grows with them, if its scores fit the work area that it may have.
constexpr int ROWS_MOST = 64;
constexpr int64_t ROWS_FLOATS = 64 << 20;
struct Plan {
    bool rows, joined;                 // rows path; in one launch
    int row_tiles, tiles, blocks;      // rows path: tiles of eight rows at a time, tiles of eight keys of a warp, blocks of keys of the longest sequence
    int64_t keys;      // of a sequence: a bound, a multiple of 128
    int tokens;        // tokens of an entry that count: a bound
    WeighTcPlan tc;
    size_t floats;
};
template <int NRT, int NG, bool FOUR, bool JOINED>
cudaError_t launch_rows(const WeighArgs& a, const b200seq_step& st, dim3 grid, int tiles, cudaStream_t cs) {
    const int smem = FOUR ? 0 : RW * RING * 2 * NG * 512;
    if (smem > 36 * 1024) {      // (beside the fragments)
        const cudaError_t e = cudaFuncSetAttribute(weigh_rows_kernel<NRT, NG, FOUR, JOINED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension, attr[1].val.clusterDim.x = JOINED ? grid.x : 1, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.gridDim = grid, cfg.blockDim = RT, cfg.dynamicSmemBytes = smem, cfg.stream = cs, cfg.attrs = attr, cfg.numAttrs = JOINED ? 2 : 1;
    cudaLaunchKernelEx(&cfg, weigh_rows_kernel<NRT, NG, FOUR, JOINED>, a, st, tiles);
    return cudaGetLastError();
}
template <int NRT, int NG, bool FOUR>
cudaError_t launch_rows(const WeighArgs& a, const b200seq_step& st, dim3 grid, int tiles, bool joined, cudaStream_t cs) {
    return joined ? launch_rows<NRT, NG, FOUR, true>(a, st, grid, tiles, cs) : launch_rows<NRT, NG, FOUR, false>(a, st, grid, tiles, cs);
}
template <int NG, bool FOUR>
cudaError_t launch_rows(const WeighArgs& a, const b200seq_step& st, dim3 grid, const Plan& p, cudaStream_t cs) {
    if (p.row_tiles == 1) return launch_rows<1, NG, FOUR>(a, st, grid, p.tiles, p.joined, cs);
    if (p.row_tiles == 2) return launch_rows<2, NG, FOUR>(a, st, grid, p.tiles, p.joined, cs);
    if (p.row_tiles == 3) return launch_rows<3, NG, FOUR>(a, st, grid, p.tiles, p.joined, cs);
    return launch_rows<4, NG, FOUR>(a, st, grid, p.tiles, p.joined, cs);
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

Plan plan_of(const b200seq_step& st, const b200seq_attn_desc& d, int last, int max_keys) {
    Plan p;
    const int64_t held = (int64_t)st.max_blocks * st.block_size;
    const int64_t keys = max_keys > 0 && max_keys < held ? max_keys : held;
    p.keys = (keys + 127) / 128 * 128;
    const int each = (st.T + st.B - 1) / (st.B > 0 ? st.B : 1), tokens = last > 0 && last < each ? last : each;      // (were all entries equally long)
    p.tokens = last > 0 && last < st.T ? last : st.T;
    const int64_t rows = (int64_t)tokens * (d.H / d.G);
    p.row_tiles = rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 24 || (rows > 32 && rows <= 48) ? 3 : 4;
    // a warp goes through as many tiles, up to sixteen, as leave four blocks an SM
    p.tiles = 1;
    while (p.tiles < MOST_TILES && p.keys * d.G * st.B / (128 * p.tiles) >= 4 * 148) p.tiles *= 2;
    p.blocks = (int)((p.keys + 64 * p.tiles - 1) / (64 * p.tiles));
    p.joined = p.blocks <= 8 && (int64_t)p.blocks * d.G * st.B <= 2 * 148;
    const int64_t floats = (int64_t)st.T * d.H * p.blocks * (64 * p.tiles + 2);
    p.rows = d.D <= 128 && rows <= ROWS_MOST && floats <= ROWS_FLOATS;
    p.tc = weigh_tc_plan(st, d.H, d.G, d.D, last, p.keys);
    const size_t lse = ((size_t)st.T * d.H + 3) / 4 * 4;      // (of the f32 tiles)
    p.floats = p.rows ? (size_t)floats : d.D <= 128 && p.tc.floats > lse ? p.tc.floats : lse;
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
    Plan p = plan_of(*st, *d, last, max_keys);
    if (!scratch || scratch_floats < p.floats || (reinterpret_cast<uintptr_t>(scratch) & 15)) return fail(B200SEQ_ERR_INVALID_ARG, "key_weights: the work area is too small or not on a 16-byte boundary");
    const bool four = kv_bits == 4;
    if (p.joined && !four && d->D > 64 && p.row_tiles == 4) p.joined = (int64_t)p.blocks * d->G * st->B <= (p.blocks <= 2 ? 2 * 148 : p.blocks <= 4 ? 256 : 240);
    if (four && (reinterpret_cast<uintptr_t>(kpool) & 15)) return fail(B200SEQ_ERR_INVALID_ARG, "key_weights: 4-bit pools start on a 16-byte boundary");
    const cudaStream_t cs = (cudaStream_t)stream;
    WeighArgs a = {};
    a.q = proj + d->q_col, a.ld = ld, a.kpool = (const float*)kpool, a.kpool4 = (const uint8_t*)kpool, a.acc = acc, a.acc_ld = acc_ld, a.slots = slots;
    a.H = d->H, a.G = d->G, a.D = d->D, a.NG = four ? kv4_groups(d->D) : 0, a.last = last, a.scale = d->scale, a.softcap = d->softcap;
    a.chunk = d->chunk, a.window = d->window, a.keep_first = d->keep_first, a.head_scale = d->head_scale, a.sink = d->sink, a.most_keys = p.keys, a.err = error_flag_dev();
    const bool wide = four || ((d->D & 3) == 0 && (reinterpret_cast<uintptr_t>(kpool) & 15) == 0);
    if (p.rows && wide) {
        a.part = scratch, a.key_blocks = p.blocks, a.key_room = (int64_t)p.blocks * 64 * p.tiles;
        const dim3 grid(p.blocks, d->G, st->B);
        cudaError_t e;
        if (four && a.NG == 1) e = launch_rows<1, true>(a, *st, grid, p, cs);
        else if (four && a.NG == 2) e = launch_rows<2, true>(a, *st, grid, p, cs);
        else if (four) e = launch_rows<4, true>(a, *st, grid, p, cs);
        else if (d->D <= 64) e = launch_rows<2, false>(a, *st, grid, p, cs);
        else e = launch_rows<4, false>(a, *st, grid, p, cs);
        if (e != cudaSuccess) return cuda_status(e, "key_weights");
        count_launch();
        if (p.joined) return 0;
        launch_chained(weigh_join_kernel, dim3((unsigned)((a.key_room + FK - 1) / FK), d->G, st->B), FT, 0, cs, a, *st, 64 * p.tiles);
        SEQ_LAUNCH_CHECK("key_weights");
        return 0;
    }
    if (weigh_tc_takes(a, four)) return weigh_tc(a, *st, p.tc, scratch, four, cs);
    a.lse = scratch;
    const int64_t tiles = ((int64_t)p.tokens * (d->H / d->G) + TR - 1) / TR, key_tiles = (p.keys + TK - 1) / TK;
    launch_chained(weigh_tile_lse_kernel, dim3((unsigned)tiles, d->G, st->B), TT, 0, cs, a, *st, (int)four);
    SEQ_LAUNCH_CHECK("key_weights");
    launch_chained(weigh_tile_sum_kernel, dim3((unsigned)key_tiles, d->G, st->B), TT, 0, cs, a, *st, (int)four);
    SEQ_LAUNCH_CHECK("key_weights");
    return 0;
}

}  // extern "C"
