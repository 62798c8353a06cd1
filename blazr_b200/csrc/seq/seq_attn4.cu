// seq_attn4.cu -- the attend step over KV pages held in 4 bits (seq_kv4.cuh has their layout), in one pass over the keys with a running maximum and sum.
//
// o = sum_j w_j v_j / sum_j w_j,  w_j = exp(z_j - max z),  z_j = scale q . k_j over the keys that a row (token, query head) sees.  With k_j = m + s u (minimum, step and
// code of a group of 32):  q . k_j = sum_groups s (q . u) + m (sum q);  with v_j = (m + 8 s) + s (u - 8):  o = sum w s (u - 8) + sum w (m + 8 s).
//
// A warp has a row tile of up to 8 rows that share a key head and walks over tiles of 32 keys, m16n8k16 products in f16 with f32 sums.  What bounds a decode
// step is the cache's bytes: 8 rows are too few for tcgen05 (128 rows a product, operands through shared memory at four times the cache's width), so the codes are
// expanded in registers, where they go straight into an operand:
//   scores  [16 x 8 keys]: the rows are A, q as two f16 numbers (22 bits): rows 0 - 7 the high parts, rows 8 - 15 the low ones, so that both products of a score meet in
//           one thread.  B is a field of the code word ANDed out: the bits 0 .. 15 as an f16 are u 2^-24 or, a field higher, u 2^-20, exactly; q takes the powers in.  s enters
//           afterwards in f32, m as one more product (the (s, m) pairs are B as they lie).
//   values  [16 x 8 columns]: the weights are A, again in two f16 parts, from the scores' own registers.  B is s (u - 8), which is an f16 number; the columns of one more
//           product are m + 8 s in two f16 parts.  (Centred, because sums of s u and of m are ten times the result: 500 keys, error 1.2e-6 with m and s summed apart.)
// So nothing is rounded but q and the weights, to 22 bits or 2^-38 of the row's largest weight, whichever is more; the rest is f32.  The tensor core cuts its f32 sums off
// instead of rounding them, 2^-21 of a sum a product, always downwards: value products are summed over 32 keys there and by rounded adds from then on (531 tokens, 2048 keys:
// error 1.3e-5 in one chain over all keys).
//
// What bounds it is instructions, not bytes: about 950 a tile of 32 keys and warp, two a cycle and SM (32 sequences of 2000 to 4000 keys, 32 query heads of 8 key heads of 128:
// 59 us, 2.1 TB/s of the cache; one of 131072 keys: 67 us, 2.5 TB/s; bytes alone 19 and 26).  One token of 500 keys, heads of 64: 5.6 us.
//
// A CTA's 8 or 4 warps share the keys of a row tile.  Few keys: so do the CTAs of a cluster, merged through distributed shared memory.  Many: the keys of all row tiles are one
// list that is dealt out evenly, and a second kernel merges the parts of row tiles that ended up in several CTAs.
#include "seq_attn4.cuh"
#include "tc_split.cuh"

namespace b200seq {

namespace {

constexpr int KT = 32;        // keys per tile: two halves of 16
constexpr int ROWS = 8;       // rows per row tile
constexpr int STAGES = 2;
// CTAs on every SM: two of 8 warps with 128 registers, or three of 4 with 168 (the plan says which)
__host__ __device__ constexpr int resident(int warps) { return warps == 8 ? 2 : 3; }
__host__ __device__ constexpr int ctas_of(int warps) { return 148 * resident(warps); }
constexpr float SLACK = 2.f;  // a maximum is raised when a score passes it by this much (base 2: weights up to 2^2)
// Weights become f16 parts times this: up to 2^15, and off by 2^-38 of the row's largest at most however small they are (f16 numbers end at 2^-24)
constexpr float WEIGHT_UP = 0x1p13f, WEIGHT_DOWN = 0x1p-13f;
constexpr float LOG2E = 1.4426950408889634f;

// d = a b + c (c may be d)
__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// two values -> f16 pair of their high parts and f16 pair of what is left (low half = a)
__device__ __forceinline__ void split16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h), lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ float par_s(uint32_t p) { return __low2float(*reinterpret_cast<const __half2*>(&p)); }
// Two codes (fields at bits 0 and 16, high: at 4 and 20) and their steps s -> s (u - 8), exactly.  A field in the mantissa of 1024 (a high one: of 64) is that number plus u; 8 and
// the number go first, which is exact, then comes the step.  (One multiply-add with -72 s would do for a high field, were that an f16 number: from s = 912 on it is not.)
__device__ __forceinline__ uint32_t centred(uint32_t x, uint32_t s_, uint32_t magic, bool high) {
    uint32_t w;
    if (high) asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(w) : "r"(x), "r"(magic));      // (x & mask) | magic
    else asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(w) : "r"(x), "r"(magic));
    const __half2 off = high ? __floats2half2_rn(-72.f, -72.f) : __floats2half2_rn(-1032.f, -1032.f);
    const __half2 d = __hmul2_rn(__hadd2_rn(*reinterpret_cast<const __half2*>(&w), off), *reinterpret_cast<const __half2*>(&s_));
    return *reinterpret_cast<const uint32_t*>(&d);
}

// steps and minima of two keys -> m + 8 s as an f16, or (low) what that rounding leaves, which is one too
__device__ __forceinline__ uint32_t centre(uint32_t s_, uint32_t m_, bool low) {
    const __half2 s = *reinterpret_cast<const __half2*>(&s_), m = *reinterpret_cast<const __half2*>(&m_), eight = __floats2half2_rn(8.f, 8.f);
    const __half2 d = __hfma2(s, eight, m), t = __hsub2_rn(d, m), e = __hadd2_rn(__hsub2_rn(m, __hsub2_rn(d, t)), __hfma2(s, eight, __hneg2(t)));
    const __half2 x = low ? e : d;
    return *reinterpret_cast<const uint32_t*>(&x);
}

// 16-byte piece i of a tile's codes in shared memory: the pieces of a 128-byte line change places with the line, so that the four keys a value load
// reads at once lie in different banks
__device__ __forceinline__ int swz(int i) { return i ^ (((i >> 3) & 3) << 1); }

// (plain loads: the compiler may move them ahead of what they do not depend on)
template <int N>
__device__ __forceinline__ void lds(const uint8_t* at, uint32_t (&x)[N]) {
    if (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(at);
        x[0] = v.x, x[1 % N] = v.y, x[2 % N] = v.z, x[3 % N] = v.w;
    } else if (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        x[0] = v.x, x[1 % N] = v.y;
    } else {
        x[0] = *reinterpret_cast<const uint32_t*>(at);
    }
}
__device__ __forceinline__ uint32_t lds16(const uint8_t* at) { return *reinterpret_cast<const uint16_t*>(at); }

// Half a tile, the 16 keys of a whole unit, into shared memory: codes (swizzled), then parameters, of keys and of values.  k, v: this lane's first piece of codes;
// par: its piece of either's parameters.  dst: the half; piece: 16 * swz(lane); par_at: where the parameters' piece goes.
template <int NK, int NV>
__device__ __forceinline__ void fetch_unit(uint32_t dst, uint32_t piece, uint32_t par_at, const uint8_t* k, const uint8_t* v, const uint8_t* par, int lane) {
    constexpr int KB = NK * 320;
#pragma unroll
    for (int n = 0; n < (NK + 1) / 2; ++n)      // (piece lane + 32 n: the same swizzle)
        if (NK > 1 || lane < 16) copy16(dst + piece + 512 * n, k + 512 * n);
#pragma unroll
    for (int n = 0; n < (NV + 1) / 2; ++n)
        if (NV > 1 || lane < 16) copy16(dst + KB + piece + 512 * n, v + 512 * n);
    if (NK + NV == 8 || lane < 4 * (NK + NV)) copy16(dst + par_at, par);
}
// the 16 keys from key0 on of one pool, from pages that a half may cross; keys behind `hi` are read from hi's row
template <int NG>
__device__ __forceinline__ void fetch_rows(uint32_t dst, const uint8_t* pool, const int32_t* bt, int bs, int key0, int hi, int g, int G, int lane, int* err) {
    for (int i = lane; i < 16 * NG * 5; i += 32) {
        const int row = i / (NG * 5), w = i - row * (NG * 5), key = min(key0 + row, hi), pg = key / bs;
        const Kv4Row at = kv4_row(kv4_page_read(bt[pg], err), key - pg * bs, bs, g, G, NG);
        if (w < NG * 4) copy4(dst + 16 * swz(row * NG + (w >> 2)) + 4 * (w & 3), pool + at.codes + 4 * w);
        else copy4(dst + NG * 256 + row * NG * 4 + 4 * (w - NG * 4), pool + at.params + 4 * (w - NG * 4));
    }
}

__device__ __forceinline__ float ld_cluster(uint32_t at, int rank) {
    uint32_t a;
    float x;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(a) : "memory");
    return x;
}

// result column `col` of (token t, head h) from a maximum, a sum and a value sum (base 2)
__device__ __forceinline__ void finish(const Attn4Args& a, int t, int h, int col, float M, float L, float acc) {
    float f = 1.f;
    if (a.sink) {   // the sink's term, under the larger of the two maxima
        const float sk = a.sink[h] * LOG2E, top = fmaxf(M, sk);
        f = tcsplit::ex2(M - top), L = fmaf(L, f, tcsplit::ex2(sk - top));
    }
    float gate = 1.f;
    if (a.gated) gate = sigmoidf_acc(a.gate[(int64_t)t * a.gld + (a.gate_elem ? (int64_t)h * a.V + col : h)]);
    store_act(a.out, a.out_dtype, ((int64_t)t * a.H + h) * a.V + col, acc * f / L * gate);
}

constexpr int MAX_TILES = 1024;             // row tiles whose keys are dealt out evenly
constexpr int HEADER = MAX_TILES + 8;       // floats of the work area in front of the parts: CTAs that have work, key tiles of a head, first key tile of every row tile

// the r-th of the step's row tiles: its entry, first token and number of tokens (0: there is none, or its positions have no pages)
__device__ __forceinline__ int row_tile(const Attn4Args& a, const b200seq_step& st, int i, int& e, int& t0, int& p0) {
    int nq = 1;
    if (st.T == st.B) {                         // (one token each, or as many entries without tokens as others have more)
        if (i >= st.T || i >= st.ent_start[st.B]) return 0;
        e = st.tok_ent[i], t0 = i;
    } else if (!attn_find_tile(st, i, a.QT, e, t0, nq)) {
        return 0;
    }
    p0 = st.tok_pos[t0];
    if (p0 < 0 || (p0 + nq - 1) / st.block_size >= st.max_blocks) {
        atomicOr(a.err, 1);
        return 0;
    }
    return nq;
}

// The keys of all row tiles and heads as one list of key tiles, head by head, dealt out evenly to the CTAs.
struct Deal {
    int64_t begin, end, total;
    int per_head;       // key tiles of one head
};
__device__ __forceinline__ int64_t deal_begin(int64_t total, int ctas, int c) { return total * c / ctas; }
__device__ __forceinline__ int deal_owner(int64_t total, int ctas, int64_t i) { return (int)(((i + 1) * ctas - 1) / total); }   // the CTA that has tile i

// first[t]: key tiles of the row tiles before t (all threads; first: shared memory, MAX_TILES + 1)
template <int WARPS>
__device__ __forceinline__ int deal_tiles(const Attn4Args& a, const b200seq_step& st, int tiles, int* first, int* sums) {
    constexpr int PER = (MAX_TILES + WARPS * 32 - 1) / (WARPS * 32);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int n[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int tile = threadIdx.x * PER + i;
        int e, t0, p0, nq = 0;
        n[i] = 0;
        if (tile < tiles) nq = row_tile(a, st, tile, e, t0, p0);
        if (nq) n[i] = KeySpan<KT>(a, p0, p0 + nq - 1).total;
        sum += n[i];
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int before = upto - sum, all = 0;
    for (int w = 0; w < WARPS; ++w) {
        before += w < warp ? sums[w] : 0;
        all += sums[w];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if ((int)threadIdx.x * PER + i < MAX_TILES) first[threadIdx.x * PER + i] = before;
        before += n[i];
    }
    if (threadIdx.x == 0) first[MAX_TILES] = all;
    __syncthreads();
    return all;
}

// Not STREAM: grid (row tiles, key heads * head blocks, cluster), a cluster's CTAs share a row tile's keys.  STREAM: ctas_of(warps) blocks, which share the keys of all row tiles evenly;
// a row tile that ends up in several leaves its parts in the work area.
template <int WARPS, int NK, int NV, bool UNITS, bool STREAM>
__global__ void __launch_bounds__(WARPS * 32, resident(WARPS)) attn4_kernel(const __grid_constant__ Attn4Args a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int KB = NK * 320, HALF = (NK + NV) * 320, STAGE = 2 * HALF, MV = 32 * NV + 4;
    auto both = [](const float (&x)[4]) { return tcsplit::add2(tcsplit::pk(x[0], x[1]), tcsplit::pk(x[2], x[3])); };      // a product's rows of high and of low parts
    __shared__ __align__(16) uint4 qfrag[(NK * 2 + 1) * 32];
    __shared__ int first[STREAM ? MAX_TILES + 1 : 1], warp_sums[STREAM ? WARPS : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int D = a.D, V = a.V, R = a.H / a.G, bs = st.block_size, rank = blockIdx.z;
    int64_t pos = 0, begin = 0, end = 1, total = 0;
    int per_head = 0;
    if (STREAM) {
        per_head = deal_tiles<WARPS>(a, st, a.tiles, first, warp_sums);
        total = (int64_t)per_head * a.heads;
        const int64_t want = (total + WARPS - 1) / WARPS;
        const int ctas = (int)(want < gridDim.x ? want : gridDim.x);
        if (blockIdx.x == 0) {
            int* head = reinterpret_cast<int*>(a.part);
            for (int i = threadIdx.x; i <= a.tiles; i += WARPS * 32) head[2 + i] = first[i < MAX_TILES ? i : MAX_TILES];
            if (threadIdx.x == 0) head[0] = ctas, head[1] = per_head;
        }
        if ((int)blockIdx.x >= ctas) return;
        begin = pos = deal_begin(total, ctas, blockIdx.x), end = deal_begin(total, ctas, blockIdx.x + 1);
    }
  do {
    int e, t0, nq, p0, unit, from = 0, to = 0;
    bool whole = false;
    if (STREAM) {
        if (pos >= end) break;
        unit = (int)(pos / per_head);
        const int at = (int)(pos - (int64_t)unit * per_head);
        int lo = 0, up = a.tiles;                     // the row tile of key tile `at`
        while (up - lo > 1) {
            const int mid = (lo + up) >> 1;
            if (first[mid] <= at) lo = mid;
            else up = mid;
        }
        nq = row_tile(a, st, lo, e, t0, p0);
        const int n = (lo + 1 < MAX_TILES ? first[lo + 1] : first[MAX_TILES]) - first[lo];
        from = at - first[lo];
        to = end - pos < n - from ? from + (int)(end - pos) : n;
        whole = from == 0 && to == n;
    } else {
        unit = blockIdx.y;
        nq = row_tile(a, st, blockIdx.x, e, t0, p0);
        if (!nq) return;                              // (all CTAs of a cluster alike)
    }
    const int g = unit / a.HB, hb = unit - g * a.HB, h0 = g * R + hb * a.Rb, nh = min(a.Rb, R - hb * a.Rb);
    const int hi = p0 + nq - 1;
    const int32_t* bt = st.block_table + (int64_t)e * st.max_blocks;
    const KeySpan<KT> span(a, p0, hi);
    const int lo_last = RowSpan(a, hi).lo;
    // ---- keys into the ring: tiles me, me + walkers, ...; the first key and the pages of a tile are looked up a tile ahead of its copies ----
    const uint32_t ring = tcpair::sa(smem) + warp * (STAGES * STAGE);
    const int walkers = STREAM ? WARPS : a.cluster * WARPS, me = STREAM ? from + warp : rank * WARPS + warp, last = STREAM ? to : span.total;
    const int nt = last > me ? (last - me + walkers - 1) / walkers : 0;
    const int upp = bs >> 4, Gv = a.G / a.vdiv;                                  // units of a page
    const uint32_t kpage = (uint32_t)(a.G * upp * (NK * 320)), vpage = (uint32_t)(Gv * upp * (NV * 320));   // (below 2^31: checked by the caller)
    const bool kpar = lane < 4 * NK;
    const uint8_t *kg = a.kpool + (int64_t)g * upp * (NK * 320), *vg = a.vpool + (int64_t)(g / a.vdiv) * upp * (NV * 320);
    const uint8_t* pg = kpar ? kg + NK * 256 + 16 * lane : vg + NV * 256 + 16 * (lane - 4 * NK);
    kg += 16 * lane, vg += 16 * lane;
    const uint32_t ppage = kpar ? kpage : vpage, piece = 16 * swz(lane), par_at = kpar ? NK * 256 + 16 * lane : KB + NV * 256 + 16 * (lane - 4 * NK);
    int key_n = span.key0(me), page0 = 0, page1 = 0;
    auto lookup = [&]() {
        if (!UNITS || key_n > hi) return;
        const int unit = key_n >> 4;
        page0 = bt[upp == 1 ? unit : unit / upp];
        if (key_n + 16 <= hi) page1 = bt[upp == 1 ? unit + 1 : (unit + 1) / upp];
    };
    auto issue = [&](int i) {      // the i-th tile of this warp, whose first key and pages have been looked up; then the next one's
        if (i < nt) {
            const uint32_t dst = ring + (i & 1) * STAGE;
            if (UNITS) {
                const int unit = key_n >> 4;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (key_n + 16 * s > hi) break;
                    const uint32_t page = (uint32_t)kv4_page_read(s ? page1 : page0, a.err);
                    const uint8_t *k = kg + (uint64_t)page * kpage, *v = vg + (uint64_t)page * vpage, *par = pg + (uint64_t)page * ppage;
                    if (upp != 1) {
                        const int u = (unit + s) % upp;
                        k += u * (NK * 320), v += u * (NV * 320), par += u * (kpar ? NK * 320 : NV * 320);
                    }
                    fetch_unit<NK, NV>(dst + s * HALF, piece, par_at, k, v, par, lane);
                }
            } else {
                for (int s = 0; s < 2 && key_n + 16 * s <= hi; ++s) {
                    fetch_rows<NK>(dst + s * HALF, a.kpool, bt, bs, key_n + 16 * s, hi, g, a.G, lane, a.err);
                    fetch_rows<NV>(dst + s * HALF + KB, a.vpool, bt, bs, key_n + 16 * s, hi, g / a.vdiv, Gv, lane, a.err);
                }
            }
            if (i + 1 < nt) key_n = span.key0(me + (i + 1) * walkers), lookup();
        }
        copies_commit();
    };
    lookup();
    int key0 = key_n;
    // ---- the rows: q as A fragments (eight neighbouring values of every group a thread), their factors and their parts against (s, m); by the first warp ----
    const int tq = r / a.Rb, hr = r - tq * a.Rb;
    const bool live = tq < nq && hr < nh;
    const RowSpan rs(a, p0 + (live ? tq : 0));
    issue(0);
    if (warp == 0) {
        const float* src = a.q + (int64_t)(t0 + tq) * a.ld + (int64_t)(h0 + hr) * D;
        float x[NK][8], mx = 0.f;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const int d = 32 * k + 8 * c;
            if (a.vec && d < D) {       // (D a multiple of 8: eight values or none)
                const float4 u = live ? ld4(src + d) : make_float4(0.f, 0.f, 0.f, 0.f), v = live ? ld4(src + d + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[k][0] = u.x, x[k][1] = u.y, x[k][2] = u.z, x[k][3] = u.w, x[k][4] = v.x, x[k][5] = v.y, x[k][6] = v.z, x[k][7] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[k][i] = live && d + i < D ? src[d + i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[k][i]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1)), mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // times a power of two that puts the largest into [2^4, 2^5); a row of zeros, denormals or infinities as it is
        const int ex = (int)(__float_as_uint(mx) >> 23);
        const bool norm = ex >= 20 && ex < 255;
        // (with the sign of the factor: what follows is scaled by its magnitude)
        float factor = a.scale;
        if (live && a.head_scale) factor *= a.head_scale[h0 + hr];
        const float up = copysignf(norm ? __uint_as_float((uint32_t)(254 - ex + 4) << 23) : 1.f, factor), down = norm ? __uint_as_float((uint32_t)(ex - 4) << 23) : 1.f;
        float mine = 0.f;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[k][i] *= up, sum += x[k][i];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1), sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            mine = k == c ? sum : mine;
#pragma unroll
            for (int s = 0; s < 2; ++s) {   // fields 0 and 4 (2 and 6) of a word, then 1 and 5 (3 and 7), which stand four bits higher
                uint4 f;
                split16(x[k][2 * s], x[k][2 * s + 4], f.x, f.y);
                split16(x[k][2 * s + 1] * 0.0625f, x[k][2 * s + 5] * 0.0625f, f.z, f.w);
                qfrag[(k * 2 + s) * 32 + lane] = f;
            }
        }
        uint4 f;
        split16(0.f, mine, f.x, f.y);   // against (s, m) of group c
        f.z = __float_as_uint(fmaxf(fabsf(factor) * (a.softcap > 0.f ? 1.f : LOG2E) * down, 1e-37f)), f.w = 0;
        qfrag[NK * 64 + lane] = f;
    }
    // where this thread's pieces lie in a half: key words of rows r and r + 8, value words and parameters of keys 2c, 2c + 1, 8 + 2c, 9 + 2c
    uint32_t ko = NK == 4 ? 16 * swz(r * 4 + c) : (NK == 2 ? 16 * swz(r * 2 + (c >> 1)) + 8 * (c & 1) : 16 * swz(r) + 4 * c), ko8 = NK == 4 ? ko + 512 : (NK == 2 ? 16 * swz((r + 8) * 2 + (c >> 1)) + 8 * (c & 1) : 16 * swz(r + 8) + 4 * c);
    uint32_t vo[4], magic64 = 0x54005400u, magic1024 = 0x64006400u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int row = 2 * c + (j & 1) + 8 * (j >> 1);
        vo[j] = KB + (NV == 4 ? 16 * swz(row * 4 + (r >> 1)) + 8 * (r & 1) : (NV == 2 ? 16 * swz(row * 2 + (r >> 2)) + 4 * (r & 3) : 16 * swz(row) + 2 * r));
    }
    asm volatile("" : "+r"(ko), "+r"(ko8), "+r"(vo[0]), "+r"(vo[1]), "+r"(vo[2]), "+r"(vo[3]), "+r"(magic64), "+r"(magic1024));   // (kept, not made again for every tile)
    __syncthreads();
    const uint2 qm = *reinterpret_cast<const uint2*>(&qfrag[NK * 64 + lane]);
    const float zf = __uint_as_float(qfrag[NK * 64 + lane].z);
    float mx = -INFINITY, l = 0.f;
    uint64_t o[NV * 4], os = 0;
#pragma unroll
    for (int k = 0; k < NV * 4; ++k) o[k] = 0;
    const float none[4] = {0.f, 0.f, 0.f, 0.f};
    const uint64_t up24 = tcsplit::pk(0x1p24f, 0x1p24f);

#pragma unroll 1
    for (int i = 0; i < nt; ++i) {
        const int key_after = key_n;      // (of the tile that is issued now)
        issue(i + 1);
        copies_wait<1>();
        __syncwarp();
        const uint8_t* const at = smem + warp * (STAGES * STAGE) + (i & 1) * STAGE;
        // ---- scores of keys key0 + 16 s + 8 n + {2c, 2c + 1}: z[4 s + 2 n + {0, 1}] ----
        float z[8];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint8_t* const ks = at + s * HALF;
            uint64_t zc[2] = {0, 0};
            uint32_t kw[2][NK], kp[4][NK];
            lds<NK>(ks + ko, kw[0]);
            if (NK == 4) lds<NK>(ks + ko + 512, kw[1]);
            else lds<NK>(ks + ko8, kw[1]);
#pragma unroll
            for (int j = 0; j < 4; ++j) lds<NK>(ks + NK * 256 + (2 * c + (j & 1) + 8 * (j >> 1)) * NK * 4, kp[j]);
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                uint4 f[2] = {qfrag[k * 64 + lane], qfrag[k * 64 + 32 + lane]};
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float acc[4];
                    const uint32_t w = kw[n][k], w8 = w >> 8;
                    mma16816(acc, f[0], w & 0x000F000Fu, w & 0x00F000F0u, none);
                    mma16816(acc, f[1], w8 & 0x000F000Fu, w8 & 0x00F000F0u, acc);
                    zc[n] = tcsplit::fma2(both(acc), tcsplit::pk(par_s(kp[2 * n][k]), par_s(kp[2 * n + 1][k])), zc[n]);
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                uint32_t b[1] = {0};
                if (c < NK) lds<1>(ks + NK * 256 + ((r + 8 * n) * NK + c) * 4, b);
                float acc[4];
                mma16816(acc, make_uint4(qm.x, qm.y, 0u, 0u), b[0], 0u, none);
                tcsplit::upk(tcsplit::fma2(zc[n], up24, both(acc)), z[4 * s + 2 * n], z[4 * s + 2 * n + 1]);
            }
        }
        if (a.softcap > 0.f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = a.softcap * LOG2E * tanhf(z[j] * zf / a.softcap);
        }
        const float zs = a.softcap > 0.f ? 1.f : zf;
        if (key0 < lo_last || key0 + KT - 1 > p0) {   // (otherwise every row sees all of the tile)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!rs.sees(key0 + 2 * c + (j & 1) + 8 * (j >> 1))) z[j] = -INFINITY;
        }
        // (rounded so that no exponent below exceeds SLACK, however large the scores: the weights' f16 parts end there)
        float tm = __fmul_ru(fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7]))), zs);
        if (__any_sync(0xffffffffu, tm > __fadd_rd(mx, SLACK))) {   // (mx = -inf: the first keys a row sees)
            tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 1)), tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 2));
            const float mn = fmaxf(mx, tm), corr = mx == -INFINITY ? 0.f : tcsplit::ex2(mx - mn);
            const uint64_t corr2 = tcsplit::pk(corr, corr);
            mx = mn, l *= corr, os = tcsplit::mul2(os, corr2);
#pragma unroll
            for (int k = 0; k < NV * 4; ++k) o[k] = tcsplit::mul2(o[k], corr2);
        }
        const float off = mx == -INFINITY ? 0.f : -mx;
        uint4 pa[2];
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = tcsplit::ex2(fmaf(z[j], zs, off));
        l += ((z[0] + z[1]) + (z[2] + z[3])) + ((z[4] + z[5]) + (z[6] + z[7]));
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] *= WEIGHT_UP;
#pragma unroll
        for (int s = 0; s < 2; ++s) split16(z[4 * s], z[4 * s + 1], pa[s].x, pa[s].y), split16(z[4 * s + 2], z[4 * s + 3], pa[s].z, pa[s].w);
        // ---- values ----
        uint32_t vw[2][4][(NV + 1) / 2], sp[2][2][NV], bp[2][2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint8_t* const vs = at + s * HALF + KB;
            uint32_t vp[4][NV], hw[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = 2 * c + (j & 1) + 8 * (j >> 1);
                lds<NV>(vs + NV * 256 + row * NV * 4, vp[j]);
                uint32_t w1[1] = {0};
                if (r < 2 * NV) lds<1>(vs + NV * 256 + (row * NV + (r >> 1)) * 4, w1);
                hw[j] = w1[0];
                if (NV == 4) lds<(NV + 1) / 2>(at + s * HALF + vo[j & 1] + 512 * (j >> 1), vw[s][j]);
                else if (NV == 2) lds<(NV + 1) / 2>(at + s * HALF + vo[j], vw[s][j]);
                else vw[s][j][0] = lds16(at + s * HALF + vo[j]);
            }
            if (key0 + 16 * s + 15 > hi) {   // whatever lies behind the last key
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (key0 + 16 * s + 2 * c + (j & 1) + 8 * (j >> 1) <= hi) continue;
                    hw[j] = 0;
#pragma unroll
                    for (int k = 0; k < NV; ++k) vp[j][k] = 0;
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                bp[s][n] = centre(__byte_perm(hw[2 * n], hw[2 * n + 1], 0x5410), __byte_perm(hw[2 * n], hw[2 * n + 1], 0x7632), r & 1);
#pragma unroll
                for (int k = 0; k < NV; ++k) sp[s][n][k] = __byte_perm(vp[2 * n][k], vp[2 * n + 1][k], 0x5410);
            }
        }
        {
            float acc[4];
            mma16816(acc, pa[0], bp[0][0], bp[0][1], none);
            mma16816(acc, pa[1], bp[1][0], bp[1][1], acc);
            os = tcsplit::add2(os, both(acc));
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int sel = (k & 1) ? 0x7632 : 0x5410;
            uint32_t x[2][2];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int n = 0; n < 2; ++n) x[s][n] = __byte_perm(vw[s][2 * n][k >> 1], vw[s][2 * n + 1][k >> 1], sel);
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                uint32_t b[2][2];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int n = 0; n < 2; ++n) b[s][n] = centred(i4 < 2 ? x[s][n] : x[s][n] >> 8, sp[s][n][k], (i4 & 1) ? magic64 : magic1024, i4 & 1);
                float acc[4];
                mma16816(acc, pa[0], b[0][0], b[0][1], none);
                mma16816(acc, pa[1], b[1][0], b[1][1], acc);
                o[4 * k + i4] = tcsplit::add2(o[4 * k + i4], both(acc));
            }
        }
        key0 = key_after;
        __syncwarp();   // the stage is refilled next
    }
    copies_wait<0>();
    // ---- the warps' parts: [warp][row][maximum, sum, -, -, values] in shared memory, over the ring; then the CTA's into the first warp's place ----
    l += __shfl_xor_sync(0xffffffffu, l, 1), l += __shfl_xor_sync(0xffffffffu, l, 2);
    float high, low;
    tcsplit::upk(os, high, low);             // of group c
    const float rest = high + low;
    __syncthreads();
    float* all = reinterpret_cast<float*>(smem);
    float* mine = all + (warp * ROWS + r) * MV;
    if (c == 0) mine[0] = mx, mine[1] = l;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const float add = __shfl_sync(0xffffffffu, rest, (lane & ~3) | k);
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            float x, y;
            tcsplit::upk(o[4 * k + i4], x, y);
            mine[4 + 32 * k + 8 * c + i4] = (x + add) * WEIGHT_DOWN, mine[4 + 32 * k + 8 * c + 4 + i4] = (y + add) * WEIGHT_DOWN;
        }
    }
    __syncthreads();
    // A warp takes a row (and row + WARPS): its maximum and sum over the warps and the factor of each one's values, then the values.
    const int cluster = STREAM ? 1 : a.cluster;
#pragma unroll 1
    for (int row = warp; row < ROWS; row += WARPS) {
        const int rt = row / a.Rb, rh = row - rt * a.Rb;
        if (rt >= nq || rh >= nh) continue;
        const float* const at = all + row * MV;
        float f[WARPS], M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, at[w * (ROWS * MV)]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float lw = at[w * (ROWS * MV) + 1];
            f[w] = lw == 0.f ? 0.f : tcsplit::ex2(at[w * (ROWS * MV)] - M);      // (0: no key that the row sees)
            L = fmaf(lw, f[w], L);
        }
        float* const pp = STREAM ? a.part + HEADER + ((int64_t)((int)blockIdx.x * 2 + (pos != begin)) * ROWS + row) * (V + 4) : nullptr;
        if (STREAM && !whole && lane == 0) pp[0] = M, pp[1] = L;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = 32 * i + lane;
            float acc = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) acc = fmaf(at[w * (ROWS * MV) + 4 + col], f[w], acc);
            if (col >= V) continue;
            if (STREAM && !whole) pp[4 + col] = acc;
            else if (cluster == 1) finish(a, t0 + rt, h0 + rh, col, M, L, acc);
            else all[row * MV + 4 + col] = acc;                                  // (the first warp's place, whose old value this thread alone has read)
        }
        __syncwarp();
        if (cluster > 1 && lane == 0) all[row * MV] = M, all[row * MV + 1] = L;
    }
    if (cluster > 1) {   // the CTAs of the cluster, each of which has a share of the rows' values
        tcpair::cluster_sync();
        const uint32_t base = tcpair::sa(all);
        const int rows = nq * nh;
        for (int i = rank * (WARPS * 32) + threadIdx.x; i < rows * V; i += cluster * (WARPS * 32)) {
            const int m = i / V, col = i - m * V, tq_ = m / nh, hr_ = m - tq_ * nh;
            const uint32_t pr = base + (tq_ * a.Rb + hr_) * MV * 4;
            float mw[8], lw[8], aw[8], top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                const bool in = w < cluster;
                mw[w] = in ? ld_cluster(pr, w) : -INFINITY, lw[w] = in ? ld_cluster(pr + 4, w) : 0.f, aw[w] = in ? ld_cluster(pr + 16 + 4 * col, w) : 0.f;
                top = fmaxf(top, mw[w]);
            }
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                const float f = lw[w] == 0.f ? 0.f : tcsplit::ex2(mw[w] - top);
                sum = fmaf(lw[w], f, sum), acc = fmaf(aw[w], f, acc);
            }
            finish(a, t0 + tq_, h0 + hr_, col, top, sum, acc);
        }
        tcpair::cluster_sync();   // nobody leaves while its shared memory is read
    }
    if (STREAM) pos += to - from, __syncthreads();    // shared memory is the next row tile's
  } while (STREAM);
}

// grid (row tiles, key heads * head blocks, blocks of 32 values), a warp a row: the parts of a row tile that several CTAs have, in order
__global__ void __launch_bounds__(ROWS * 32) attn4_gather_kernel(const __grid_constant__ Attn4Args a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    __shared__ float factor[ROWS][ctas_of(4)];
    const int* head = reinterpret_cast<const int*>(a.part);
    const int ctas = head[0], per_head = head[1], n = head[3 + blockIdx.x] - head[2 + blockIdx.x];
    if (n == 0) return;
    const int64_t total = (int64_t)per_head * a.heads, u0 = (int64_t)blockIdx.y * per_head + head[2 + blockIdx.x];
    const int c0 = deal_owner(total, ctas, u0), c1 = deal_owner(total, ctas, u0 + n - 1);
    if (c0 == c1) return;                             // one CTA had it all
    int e, t0, p0;
    const int nq = row_tile(a, st, blockIdx.x, e, t0, p0);
    const int R = a.H / a.G, g = blockIdx.y / a.HB, hb = blockIdx.y - g * a.HB, h0 = g * R + hb * a.Rb, nh = min(a.Rb, R - hb * a.Rb);
    const int row = threadIdx.x >> 5, lane = threadIdx.x & 31, tq = row / a.Rb, hr = row - tq * a.Rb, step = a.V + 4;
    if (tq >= nq || hr >= nh) return;
    // a CTA's part of this row tile lies in its first place if its share begins there or before, else in its second
    const int64_t pitch = (int64_t)2 * ROWS * step;
    const float* const parts = a.part + HEADER + c0 * pitch + (int64_t)row * step;
    const float* const own = deal_begin(total, ctas, c0) != u0 ? parts + (int64_t)ROWS * step : parts;      // c0's
    const int np = c1 - c0 + 1;
    auto part = [&](int i) { return i ? parts + i * pitch : own; };
    float M = -INFINITY, L = 0.f;
    for (int i = lane; i < np; i += 32) M = fmaxf(M, part(i)[0]);
    M = warp_max(M);
    for (int i = lane; i < np; i += 32) {
        const float l = part(i)[1], f = l == 0.f ? 0.f : tcsplit::ex2(part(i)[0] - M);      // (0: no key that the row sees)
        factor[row][i] = f;
        L = fmaf(l, f, L);
    }
    L = warp_sum(L);
    __syncwarp();
    const int col = blockIdx.z * 32 + lane;
    if (col >= a.V) return;
    float acc = own[4 + col] * factor[row][0];
#pragma unroll 8
    for (int i = 1; i < np; ++i) acc = fmaf(parts[i * pitch + 4 + col], factor[row][i], acc);
    finish(a, t0 + tq, h0 + hr, col, M, L, acc);
}

// grid (T, H): the parts that the tensor-core kernel leaves of one (token, head), in order
__global__ void attn4_merge_kernel(const __grid_constant__ Attn4Args a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    const int t = blockIdx.x, h = blockIdx.y, n = a.parts, step = a.V + 4;
    const float* pp = a.part + ((int64_t)t * a.H + h) * n * step;
    float M = -INFINITY, L = 0.f;
    if (t >= st.ent_start[st.B] || pp[1] < 0.f) return;      // nobody's row; a row whose positions have no pages
    for (int w = 0; w < n; ++w) M = fmaxf(M, pp[w * step]);
    for (int w = 0; w < n; ++w)
        if (pp[w * step + 1] != 0.f) L = fmaf(pp[w * step + 1], tcsplit::ex2(pp[w * step] - M), L);
    for (int col = threadIdx.x; col < a.V; col += blockDim.x) {
        float acc = 0.f;
        for (int w = 0; w < n; ++w)
            if (pp[w * step + 1] != 0.f) acc = fmaf(pp[w * step + 4 + col], tcsplit::ex2(pp[w * step] - M), acc);
        finish(a, t, h, col, M, L, acc);
    }
}

template <int WARPS, int NK, int NV, bool UNITS, bool STREAM>
cudaError_t launch(const Attn4Args& a, const b200seq_step& st, dim3 grid, cudaStream_t cs) {
    constexpr int ring = WARPS * STAGES * 2 * (NK + NV) * 320, parts = WARPS * ROWS * (32 * NV + 4) * 4, smem = ring > parts ? ring : parts;
    const auto kernel = attn4_kernel<WARPS, NK, NV, UNITS, STREAM>;
    static bool ready[16] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 16 || !ready[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 16) ready[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension, attr[1].val.clusterDim.x = attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = a.cluster;
    cfg.gridDim = grid, cfg.blockDim = WARPS * 32, cfg.dynamicSmemBytes = smem, cfg.stream = cs, cfg.attrs = attr, cfg.numAttrs = a.cluster > 1 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kernel, a, st);
    return e != cudaSuccess ? e : cudaGetLastError();
}
// the most keys a token can see: what the block tables hold, or the fewer that the caller names (a bound to plan by; nothing goes wrong with more of them)
int64_t most_keys(const b200seq_step& st, const b200seq_attn_desc& d, int max_keys, int tokens) {
    int64_t keys = (int64_t)st.max_blocks * st.block_size;
    if (max_keys > 0 && max_keys < keys) keys = max_keys;
    if (d.chunk > 0 && d.chunk < keys) keys = d.chunk;
    if (d.window > 0 && (int64_t)d.window + d.keep_first + tokens < keys) keys = (int64_t)d.window + d.keep_first + tokens;
    return keys;
}
// How the keys of a step are shared.  Row tiles and heads go to a CTA each, or to a cluster of up to 8 while there are CTAs for all and keys for all their warps.  Few of them
// with many keys are dealt out evenly, with a second launch for those that several CTAs have; that costs about 8 us a row tile begun and 5 for the launch (32 sequences, 256
// row tiles and heads: 65 us dealt, 55 not; one sequence of 40000 keys, heads of 64: 26 dealt, 33 in a cluster; of 131072, heads of 128: 66 and 110).  CTAs have the 8 or 4 warps whose last wave is the fuller one (256 row tiles
// and heads of 128, 3000 keys: 55 us with 8, 77 with 4; 16 x 5 tokens, 384 of 64, 1500 keys: 29 with 8, 24 with 4); the small ones for heads of up to 64 where that is the same.
struct Plan {
    int64_t tiles, real;     // row tiles: upper bound; as many as there are if all entries are equally long
    int heads, cluster, warps, ctas;
    bool dealt;
};
// us of row tiles with kt key tiles each that have CTAs of their own, or whose keys are dealt out
double shared_us(const Plan& p, bool small, double kt) {
    const double waves = (double)p.real * p.heads * p.cluster / p.ctas, share = kt / (p.warps * p.cluster), least = p.warps == 4 ? 0.4 : (small ? 0.85 : 0.53);
    const double tile = (small ? 1.5 : 3.6) * (waves < least ? least : (waves < 1.0 ? waves : 1.0));
    return (waves < 1.0 ? 1.0 : waves) * ((small ? 4.0 : 5.0) + tile * (share < 1.0 ? 1.0 : share)) + 2.0;
}
double dealt_us(bool small, double units, double kt) { return small ? 18.0 + units * kt / 1200.0 : 15.5 + units * kt / 645.0; }
Plan plan(const b200seq_step& st, const b200seq_attn_desc& d, int max_keys) {
    Plan p;
    const int R = d.H / d.G, Rb = R < ROWS ? R : ROWS, QT = ROWS / Rb;
    p.heads = d.G * ((R + Rb - 1) / Rb);
    p.tiles = st.T == st.B ? st.T : ((int64_t)st.T + QT - 1) / QT + st.B;
    const int64_t each = ((int64_t)st.T + st.B - 1) / st.B;
    p.real = st.B * ((each + QT - 1) / QT);
    const int64_t units = p.real * p.heads, key_tiles = (most_keys(st, d, max_keys, QT) + KT - 1) / KT;
    const bool small = d.D <= 64 && d.V <= 64;
    double best = -1.0;
    for (int warps : {small ? 4 : 8, small ? 8 : 4}) {
        const int ctas = ctas_of(warps);
        int64_t want = ctas / units, most = (key_tiles + warps - 1) / warps;
        want = want < most ? want : most;
        const int cluster = want >= 8 ? 8 : (want >= 4 ? 4 : (want >= 2 ? 2 : 1));
        const int64_t n = units * cluster, waves = (n + ctas - 1) / ctas;
        const double full = (double)n / (double)(waves * ctas);
        if (full > best * 1.05) best = full, p.warps = warps, p.ctas = ctas, p.cluster = cluster;
    }
    p.dealt = st.block_size % 16 == 0 && p.tiles <= MAX_TILES && units * p.cluster * 2 <= p.ctas && dealt_us(small, (double)units, (double)key_tiles) + 2.0 < shared_us(p, small, (double)key_tiles);
    if (p.dealt) p.cluster = 1, p.warps = small ? 4 : 8, p.ctas = ctas_of(p.warps);
    return p;
}
template <int NK, int NV>
cudaError_t launch_form(const Attn4Args& a, const b200seq_step& st, dim3 grid, const Plan& p, cudaStream_t cs) {
    if (st.block_size % 16) return p.warps == 8 ? launch<8, NK, NV, false, false>(a, st, grid, cs) : launch<4, NK, NV, false, false>(a, st, grid, cs);
    if (p.dealt) return launch<(NK == 4 || NV == 4 ? 8 : 4), NK, NV, true, true>(a, st, grid, cs);
    return p.warps == 8 ? launch<8, NK, NV, true, false>(a, st, grid, cs) : launch<4, NK, NV, true, false>(a, st, grid, cs);
}
template <int NK>
cudaError_t launch_values(int nv, const Attn4Args& a, const b200seq_step& st, dim3 grid, const Plan& p, cudaStream_t cs) {
    return nv == 1 ? launch_form<NK, 1>(a, st, grid, p, cs) : (nv == 2 ? launch_form<NK, 2>(a, st, grid, p, cs) : launch_form<NK, 4>(a, st, grid, p, cs));
}
// Which kernel is the faster one, from the key tiles a CTA has at most.  us, fitted to measured steps.  146 steps of 1 to 288 tokens have been timed with each of the two (a table
// in profiles/kv4_choice.txt): the choice is 18 % behind the faster one at most (8 x 16 tokens behind 1000, heads of 64), in 143 of them 3 % or less.  Here (shared_us, dealt_us): a wave of CTAs takes 4 (5 with heads above 64) and 1.5 (3.6) a key tile of 32 and warp, down to 0.6 (four
// warps) or 1.3 (1.9) where a CTA has an SM to itself; keys that are dealt out 18 (15.5), and 1200 (645) key tiles a us.  On the tensor cores: 7.5 (9; f32 11) a CTA
// and 0.8 (0.75; f32 1.4) a key tile of 64, 4 more for keys in several parts.  Measured, us, here / there, 32 query heads of 8 key heads of 64 (of 128):
//   1 x 64 tokens                6 /  8 ( 8 / 10)     16 x 9 behind 1500   45 / 29 (67 / 32)     32 x 2 behind 2000   34 / 65 (45 / 71)
//   1 x 32 behind 4000          23 / 23 (35 / 25)      4 x 8 behind 8000   41 / 36 (62 / 41)      4 x 64 behind 300   28 / 13 (40 / 14)
bool tc_is_faster(const b200seq_step& st, const b200seq_attn_desc& d, int max_keys, const Plan& p, const Attn4TcPlan& tp, bool f32) {
    const bool small = d.D <= 64 && d.V <= 64;
    const double keys = (double)most_keys(st, d, max_keys, 0), kt = (keys + KT - 1) / KT;
    const double here = p.dealt ? dealt_us(small, (double)p.real * p.heads, kt) : shared_us(p, small, kt);
    const double set_up = small ? 7.5 : (f32 ? 11.0 : 9.0), each = small ? 0.8 : (f32 ? 1.4 : 0.75);
    const int64_t tc_waves = (tp.real * tp.parts + 147) / 148;
    const double there = (double)tc_waves * (set_up + each * (keys / 64.0 / tp.parts + 0.5)) + 2.0 + (tp.parts > 1 ? 4.0 : 0.0);
    return there < here;
}
size_t plan_floats(const Plan& p, int V) { return p.dealt ? (size_t)HEADER + (size_t)p.ctas * 2 * ROWS * (V + 4) : 0; }

}  // namespace

}  // namespace b200seq

using namespace b200seq;

extern "C" {

size_t b200seq_attn_kv4_scratch_floats(const b200seq_step* st, const b200seq_attn_desc* d, int max_keys) {
    if (!st || !d || st->T < 1 || st->B < 1 || st->block_size < 1 || st->max_blocks < 1 || d->H < 1 || d->G < 1 || d->H % d->G || d->V < 1) return 0;
    const Plan p = plan(*st, *d, max_keys);
    size_t need = plan_floats(p, d->V);
    if (attn4_tc_takes(d->D, d->V)) {
        const Attn4TcPlan tp = attn4_tc_plan(*st, d->H, d->G, d->D, d->V, most_keys(*st, *d, max_keys, 0));
        if (tp.parts > 1 && tc_is_faster(*st, *d, max_keys, p, tp, false)) {   // (chosen for f32 results: chosen for bf16 ones too)
            const size_t tc = (size_t)st->T * d->H * tp.parts * (d->V + 4);
            need = tc > need ? tc : need;
        }
    }
    return need;
}

int b200seq_attn_kv4(const float* proj, int64_t ld, const b200seq_step* st, const b200seq_attn_desc* d, const void* kpool, const void* vpool, void* out, int out_dtype,
                     float* scratch, size_t scratch_floats, int max_keys, void* stream) {
    if (int rc = attn_desc_check(d, "attn_kv4")) return rc;
    if (!st || st->T < 0 || st->B < 0 || st->block_size < 1 || st->max_blocks < 0) return fail(B200SEQ_ERR_INVALID_ARG, "attn_kv4: bad step");
    if (!proj || !kpool || !vpool || !out || (st->T > 0 && (!st->tok_ent || !st->tok_pos || !st->ent_start || !st->block_table)))
        return fail(B200SEQ_ERR_INVALID_ARG, "attn_kv4: bad arguments");
    if (out_dtype != B200SEQ_F32 && out_dtype != B200SEQ_BF16) return fail(B200SEQ_ERR_INVALID_ARG, "attn_kv4: results are f32 or bf16");
    if (d->pool > 0 || d->latent_v || d->krot || d->ctx_rows || d->kv_ld > 0 || (d->kd > 0 && d->kd < d->D))
        return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: a 4-bit cache holds plain keys and values (no pooled blocks, no latents)");
    if (d->D > KV4_MAX_DIM || d->V > KV4_MAX_DIM) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: heads of up to %d values", KV4_MAX_DIM);
    if ((reinterpret_cast<uintptr_t>(kpool) | reinterpret_cast<uintptr_t>(vpool)) & 15) return fail(B200SEQ_ERR_INVALID_ARG, "attn_kv4: pools start on a 16-byte boundary");
    if (st->block_size > 1 << 16) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: pages of up to 65536 tokens");
    const int64_t page = (int64_t)20 * st->block_size * d->G * kv4_groups(d->D > d->V ? d->D : d->V);
    if (page > 0x7fffffff) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: pages of up to 2 GiB");
    if (st->T == 0) return 0;
    if (st->B < 1) return fail(B200SEQ_ERR_INVALID_ARG, "attn_kv4: tokens without an entry");
    const bool gated = d->gate_col >= 0;
    const int R = d->H / d->G;
    Attn4Args a = {};
    a.q = proj + d->q_col, a.ld = ld, a.kpool = (const uint8_t*)kpool, a.vpool = (const uint8_t*)vpool;
    a.H = d->H, a.G = d->G, a.D = d->D, a.V = d->V, a.vdiv = d->vg > 0 ? d->G / d->vg : 1;
    a.Rb = R < ROWS ? R : ROWS, a.HB = (R + a.Rb - 1) / a.Rb, a.QT = ROWS / a.Rb;
    a.scale = d->scale, a.chunk = d->chunk, a.window = d->window, a.keep_first = d->keep_first, a.head_scale = d->head_scale, a.sink = d->sink;
    a.gate = d->gate ? d->gate : proj + (gated ? d->gate_col : 0), a.gld = d->gate ? d->gate_ld : ld, a.gated = gated, a.gate_elem = gated && d->gate_elem;
    a.vec = ((ld | d->q_col) & 3) == 0 && d->D % 8 == 0 && (reinterpret_cast<uintptr_t>(proj) & 15) == 0;
    a.softcap = d->softcap, a.out = out, a.out_dtype = out_dtype, a.err = error_flag_dev();
    cudaStream_t cs = (cudaStream_t)stream;
    if (d->H > 65535) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: too many heads");
    Plan p = plan(*st, *d, max_keys);
    Attn4TcPlan tp = attn4_tc_plan(*st, d->H, d->G, d->D, d->V, most_keys(*st, *d, max_keys, 0));
    if (a.vec && attn4_tc_takes(d->D, d->V) && tc_is_faster(*st, *d, max_keys, p, tp, out_dtype == B200SEQ_F32)) {
        if (tp.parts > 1 && (!scratch || scratch_floats < (size_t)st->T * d->H * tp.parts * (d->V + 4))) tp.parts = 1;
        if ((int64_t)d->G * tp.HB * tp.tiles > 0x7fffffff) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: too many heads or tokens");
        a.part = scratch, a.parts = tp.parts;
        const cudaError_t e = attn4_tc_launch(a, *st, tp, cs);
        if (e != cudaSuccess) return cuda_status(e, "attn_kv4");
        count_launch();
        if (tp.parts > 1) {
            launch_chained(attn4_merge_kernel, dim3(st->T, d->H), d->V <= 64 ? 64 : 128, 0, cs, a, *st);
            SEQ_LAUNCH_CHECK("attn_kv4 merge");
        }
        return 0;
    }
    if (p.dealt && (!scratch || scratch_floats < plan_floats(p, d->V))) p.dealt = false;
    if (p.heads > 65535 || p.tiles > 0x7fffffff) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: too many heads or tokens");
    a.cluster = p.cluster, a.parts = 1, a.part = scratch, a.tiles = (int)p.tiles, a.heads = p.heads;
    const dim3 grid = p.dealt ? dim3((unsigned)p.ctas) : dim3((unsigned)p.tiles, (unsigned)p.heads, (unsigned)p.cluster);
    const int nk = kv4_groups(d->D), nv = kv4_groups(d->V);
    const cudaError_t e = nk == 1 ? launch_values<1>(nv, a, *st, grid, p, cs) : (nk == 2 ? launch_values<2>(nv, a, *st, grid, p, cs) : launch_values<4>(nv, a, *st, grid, p, cs));
    if (e != cudaSuccess) return cuda_status(e, "attn_kv4");
    count_launch();
    if (p.dealt) {
        launch_chained(attn4_gather_kernel, dim3((unsigned)p.tiles, (unsigned)p.heads, (unsigned)((d->V + 31) / 32)), ROWS * 32, 0, cs, a, *st);
        SEQ_LAUNCH_CHECK("attn_kv4 gather");
    }
    return 0;
}

}  // extern "C"
