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
// So nothing is rounded but q and the weights to 22 bits; the rest is f32.  The tensor core cuts its f32 sums off instead of rounding them, 2^-21 of a sum a product, always
// downwards: value products are summed over 32 keys there and by rounded adds from then on (531 tokens, 2048 keys: error 1.3e-5 in one chain over all keys).
//
// Keys are dealt to the 8 warps of a CTA, to the CTAs of a cluster (merged through distributed shared memory) and, where that leaves SMs idle, to several clusters
// (merged by a second kernel through the work area).
#include "seq_attn4.cuh"
#include "tc_split.cuh"

namespace b200seq {

namespace {

constexpr int KT = 32;        // keys per tile: two halves of 16
constexpr int ROWS = 8;       // rows per row tile
constexpr int WARPS = 8;
constexpr int STAGES = 2;
constexpr float SLACK = 8.f;  // a maximum is raised when a score passes it by this much (weights up to 2^8, where f16 parts are as good)
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
__device__ __forceinline__ float par_s(uint32_t p) { return __half2float(__ushort_as_half((uint16_t)p)); }
// two codes (fields at bits 0 and 16, high: at 4 and 20) and their steps -> s (u - 8), exactly: 0x6400 | u is 1024 + u, with a field of 16 u divided out
__device__ __forceinline__ uint32_t centred(uint32_t x, uint32_t s, bool high) {
    const uint32_t w = (x & (high ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    const __half2 u = high ? __hfma2(h, __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-72.f, -72.f)) : __hadd2_rn(h, __floats2half2_rn(-1032.f, -1032.f));
    const __half2 d = __hmul2_rn(u, *reinterpret_cast<const __half2*>(&s));
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

template <int N>
__device__ __forceinline__ void lds(uint32_t at, uint32_t (&x)[N]) {
    if (N == 4) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[N > 2 ? 2 : 0]), "=r"(x[N > 3 ? 3 : 0]) : "r"(at) : "memory");
    else if (N == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[N > 1 ? 1 : 0]) : "r"(at) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x[0]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t lds16(uint32_t at) {
    uint16_t x;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at) : "memory");
    return x;
}

// half a tile, the 16 keys from key0 on, into shared memory: codes (swizzled), then parameters.  Keys behind `hi` are read from hi's row, or, in whole units, from the
// rest of its page.
template <int NG, bool UNITS>
__device__ __forceinline__ void fetch(uint32_t dst, const uint8_t* pool, const int32_t* bt, int bs, int key0, int hi, int g, int G, int lane) {
    if (UNITS) {
        const int pg = key0 / bs;
        const uint8_t* src = pool + ((int64_t)bt[pg] * G + g) * (int64_t)(bs * NG * 20) + (key0 - pg * bs) * (NG * 20);
#pragma unroll
        for (int i = lane; i < NG * 20; i += 32) copy16(dst + 16 * (i < NG * 16 ? swz(i) : i), src + 16 * i);
    } else {
        for (int i = lane; i < 16 * NG * 5; i += 32) {
            const int row = i / (NG * 5), w = i - row * (NG * 5), key = min(key0 + row, hi), pg = key / bs;
            const Kv4Row at = kv4_row(bt[pg], key - pg * bs, bs, g, G, NG);
            if (w < NG * 4) copy4(dst + 16 * swz(row * NG + (w >> 2)) + 4 * (w & 3), pool + at.codes + 4 * w);
            else copy4(dst + NG * 256 + row * NG * 4 + 4 * (w - NG * 4), pool + at.params + 4 * (w - NG * 4));
        }
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

// grid (row tiles * parts, key heads * head blocks, 1), clusters along z: (row tile, part, rank) share nothing but the merge
template <int NK, int NV, bool UNITS>
__global__ void __launch_bounds__(WARPS * 32, 2) attn4_kernel(const __grid_constant__ Attn4Args a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int KB = NK * 320, HALF = (NK + NV) * 320, STAGE = 2 * HALF, MV = 32 * NV + 4;
    __shared__ __align__(16) uint4 qfrag[NK * 2 * 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int D = a.D, V = a.V, R = a.H / a.G, bs = st.block_size, rank = blockIdx.z;
    const int tile_no = blockIdx.x / a.parts, seg = blockIdx.x - tile_no * a.parts;
    int e, t0, nq;
    if (st.T == st.B) e = t0 = tile_no, nq = 1;
    else if (!attn_find_tile(st, tile_no, a.QT, e, t0, nq)) return;      // (all CTAs of a cluster alike)
    const int g = blockIdx.y / a.HB, hb = blockIdx.y - g * a.HB, h0 = g * R + hb * a.Rb, nh = min(a.Rb, R - hb * a.Rb);
    const int p0 = st.tok_pos[t0], hi = p0 + nq - 1;
    const int32_t* bt = st.block_table + (int64_t)e * st.max_blocks;
    if (p0 < 0 || hi / bs >= st.max_blocks) {
        if (threadIdx.x == 0) atomicOr(a.err, 1);
        return;
    }
    const KeySpan<KT> span(a, p0, hi);
    const int lo_last = RowSpan(a, hi).lo;
    // ---- keys into the ring ----
    const uint32_t ring = tcpair::sa(smem) + warp * (STAGES * STAGE);
    const int walkers = a.parts * a.cluster * WARPS, me = (seg * a.cluster + rank) * WARPS + warp;
    const int nt = span.total > me ? (span.total - me + walkers - 1) / walkers : 0;
    auto issue = [&](int i) {
        if (i < nt) {
            const int key0 = span.key0(me + i * walkers);
            const uint32_t dst = ring + (i & 1) * STAGE;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (key0 + 16 * s > hi) break;
                fetch<NK, UNITS>(dst + s * HALF, a.kpool, bt, bs, key0 + 16 * s, hi, g, a.G, lane);
                fetch<NV, UNITS>(dst + s * HALF + KB, a.vpool, bt, bs, key0 + 16 * s, hi, g / a.vdiv, a.G / a.vdiv, lane);
            }
        }
        copies_commit();
    };
    issue(0);
    // ---- this thread's row: q as A fragments (eight neighbouring values of every group), its factor and what it sees ----
    const int tq = r / a.Rb, hr = r - tq * a.Rb;
    const bool live = tq < nq && hr < nh;
    const RowSpan rs(a, p0 + (live ? tq : 0));
    float zf;
    uint32_t qm[4] = {0u, 0u, 0u, 0u};
    {
        const float* src = a.q + (int64_t)(t0 + tq) * a.ld + (int64_t)(h0 + hr) * D;
        float x[NK][8], mx = 0.f;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = 32 * k + 8 * c + i;
                x[k][i] = live && d < D ? src[d] : 0.f;
                mx = fmaxf(mx, fabsf(x[k][i]));
            }
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
            if (warp == 0) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {   // fields 0 and 4 (2 and 6) of a word, then 1 and 5 (3 and 7), which stand four bits higher
                    uint4 f;
                    split16(x[k][2 * s], x[k][2 * s + 4], f.x, f.y);
                    split16(x[k][2 * s + 1] * 0.0625f, x[k][2 * s + 5] * 0.0625f, f.z, f.w);
                    qfrag[(k * 2 + s) * 32 + lane] = f;
                }
            }
        }
        split16(0.f, mine, qm[0], qm[1]);   // against (s, m) of group c
        zf = fmaxf(fabsf(factor) * (a.softcap > 0.f ? 1.f : LOG2E) * down, 1e-37f);
    }
    __syncthreads();
    float mx = -INFINITY, l = 0.f;
    uint64_t o[NV * 4], os = 0;
#pragma unroll
    for (int k = 0; k < NV * 4; ++k) o[k] = 0;
    const float none[4] = {0.f, 0.f, 0.f, 0.f};
    const uint64_t up24 = tcsplit::pk(0x1p24f, 0x1p24f);

#pragma unroll 1
    for (int i = 0; i < nt; ++i) {
        issue(i + 1);
        copies_wait<1>();
        __syncwarp();
        const uint32_t at = ring + (i & 1) * STAGE;
        const int key0 = span.key0(me + i * walkers);
        // ---- scores of keys key0 + 16 s + 8 n + {2c, 2c + 1}: z[4 s + 2 n + {0, 1}] ----
        float z[8];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t ks = at + s * HALF;
            uint64_t zc[2] = {0, 0};
            uint32_t kw[2][NK], kp[4][NK];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int row = r + 8 * n;
                lds<NK>(ks + (NK == 4 ? 16 * swz(row * 4 + c) : (NK == 2 ? 16 * swz(row * 2 + (c >> 1)) + 8 * (c & 1) : 16 * swz(row) + 4 * c)), kw[n]);
            }
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
                    zc[n] = tcsplit::fma2(tcsplit::add2(tcsplit::pk(acc[0], acc[1]), tcsplit::pk(acc[2], acc[3])), tcsplit::pk(par_s(kp[2 * n][k]), par_s(kp[2 * n + 1][k])), zc[n]);
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                uint32_t b[1] = {0};
                if (c < NK) lds<1>(ks + NK * 256 + ((r + 8 * n) * NK + c) * 4, b);
                float acc[4];
                mma16816(acc, make_uint4(qm[0], qm[1], 0u, 0u), b[0], 0u, none);
                tcsplit::upk(tcsplit::fma2(zc[n], up24, tcsplit::add2(tcsplit::pk(acc[0], acc[1]), tcsplit::pk(acc[2], acc[3]))), z[4 * s + 2 * n], z[4 * s + 2 * n + 1]);
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
        float tm = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7]))) * zs;
        if (__any_sync(0xffffffffu, tm > mx + SLACK)) {   // (mx = -inf: the first keys a row sees)
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
        for (int s = 0; s < 2; ++s) split16(z[4 * s], z[4 * s + 1], pa[s].x, pa[s].y), split16(z[4 * s + 2], z[4 * s + 3], pa[s].z, pa[s].w);
        // ---- values ----
        uint32_t vw[2][4][(NV + 1) / 2], sp[2][2][NV], bp[2][2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t vs = at + s * HALF + KB;
            uint32_t vp[4][NV], hw[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = 2 * c + (j & 1) + 8 * (j >> 1);
                lds<NV>(vs + NV * 256 + row * NV * 4, vp[j]);
                uint32_t w1[1] = {0};
                if (r < 2 * NV) lds<1>(vs + NV * 256 + (row * NV + (r >> 1)) * 4, w1);
                hw[j] = w1[0];
                if (NV == 4) lds<(NV + 1) / 2>(vs + 16 * swz(row * 4 + (r >> 1)) + 8 * (r & 1), vw[s][j]);
                else if (NV == 2) lds<(NV + 1) / 2>(vs + 16 * swz(row * 2 + (r >> 2)) + 4 * (r & 3), vw[s][j]);
                else vw[s][j][0] = lds16(vs + 16 * swz(row) + 2 * r);
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
            os = tcsplit::add2(os, tcsplit::add2(tcsplit::pk(acc[0], acc[1]), tcsplit::pk(acc[2], acc[3])));
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
                    for (int n = 0; n < 2; ++n) b[s][n] = centred(i4 < 2 ? x[s][n] : x[s][n] >> 8, sp[s][n][k], i4 & 1);
                float acc[4];
                mma16816(acc, pa[0], b[0][0], b[0][1], none);
                mma16816(acc, pa[1], b[1][0], b[1][1], acc);
                o[4 * k + i4] = tcsplit::add2(o[4 * k + i4], tcsplit::add2(tcsplit::pk(acc[0], acc[1]), tcsplit::pk(acc[2], acc[3])));
            }
        }
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
            mine[4 + 32 * k + 8 * c + i4] = x + add, mine[4 + 32 * k + 8 * c + 4 + i4] = y + add;
        }
    }
    __syncthreads();
    const int rows = nq * nh, cluster = a.cluster;
    // what several places hold for one row and column, at(w) the w-th one's (maximum, sum, value)
    auto merge = [](int n, auto&& at, float& M, float& L, float& acc) {
        M = -INFINITY, L = acc = 0.f;
        for (int w = 0; w < n; ++w) M = fmaxf(M, at(w, 0));
        for (int w = 0; w < n; ++w) {
            const float lw = at(w, 1);
            if (lw == 0.f) continue;          // no key that the row sees
            const float f = tcsplit::ex2(at(w, 0) - M);
            L = fmaf(lw, f, L), acc = fmaf(at(w, 2), f, acc);
        }
    };
    if (cluster == 1 && a.parts == 1) {
        for (int i = threadIdx.x; i < rows * V; i += WARPS * 32) {
            const int m = i / V, col = i - m * V, tq_ = m / nh, hr_ = m - tq_ * nh;
            const float* pr = all + (tq_ * a.Rb + hr_) * MV;
            float M, L, acc;
            merge(WARPS, [&](int w, int what) { return pr[w * (ROWS * MV) + (what < 2 ? what : 4 + col)]; }, M, L, acc);
            finish(a, t0 + tq_, h0 + hr_, col, M, L, acc);
        }
        return;
    }
    float* cta = all + WARPS * ROWS * MV;     // [row][maximum, sum, -, -, values]
    for (int i = threadIdx.x; i < ROWS * V; i += WARPS * 32) {
        const int m = i / V, col = i - m * V;
        const float* pr = all + m * MV;
        float M, L, acc;
        merge(WARPS, [&](int w, int what) { return pr[w * (ROWS * MV) + (what < 2 ? what : 4 + col)]; }, M, L, acc);
        if (col == 0) cta[m * MV] = M, cta[m * MV + 1] = L;
        cta[m * MV + 4 + col] = acc;
    }
    if (cluster > 1) tcpair::cluster_sync();
    else __syncthreads();
    const uint32_t base = tcpair::sa(cta);
    for (int i = rank * (WARPS * 32) + threadIdx.x; i < rows * V; i += cluster * (WARPS * 32)) {
        const int m = i / V, col = i - m * V, tq_ = m / nh, hr_ = m - tq_ * nh, t = t0 + tq_, h = h0 + hr_;
        const uint32_t pr = base + (tq_ * a.Rb + hr_) * MV * 4;
        float M, L, acc;
        merge(cluster, [&](int w, int what) { return ld_cluster(pr + 4 * (what < 2 ? what : 4 + col), w); }, M, L, acc);
        if (a.parts == 1) {
            finish(a, t, h, col, M, L, acc);
        } else {
            float* pp = a.part + (((int64_t)t * a.H + h) * a.parts + seg) * (V + 4);
            if (col == 0) pp[0] = M, pp[1] = L;
            pp[4 + col] = acc;
        }
    }
    if (cluster > 1) tcpair::cluster_sync();  // nobody leaves while its shared memory is read
}

// grid (T, H): the clusters' parts of one (token, head), in order
__global__ void attn4_merge_kernel(const __grid_constant__ Attn4Args a) {
    chain_enter();
    const int t = blockIdx.x, h = blockIdx.y, n = a.parts, step = a.V + 4;
    const float* pp = a.part + ((int64_t)t * a.H + h) * n * step;
    float M = -INFINITY, L = 0.f;
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

template <int NK, int NV, bool UNITS>
cudaError_t launch(const Attn4Args& a, const b200seq_step& st, dim3 grid, cudaStream_t cs) {
    constexpr int ring = WARPS * STAGES * 2 * (NK + NV) * 320, parts = (WARPS + 1) * ROWS * (32 * NV + 4) * 4, smem = ring > parts ? ring : parts;
    const auto kernel = attn4_kernel<NK, NV, UNITS>;
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
template <int NK, int NV>
cudaError_t launch_units(const Attn4Args& a, const b200seq_step& st, dim3 grid, cudaStream_t cs) {
    return st.block_size % 16 == 0 ? launch<NK, NV, true>(a, st, grid, cs) : launch<NK, NV, false>(a, st, grid, cs);
}
template <int NK>
cudaError_t launch_values(int nv, const Attn4Args& a, const b200seq_step& st, dim3 grid, cudaStream_t cs) {
    return nv == 1 ? launch_units<NK, 1>(a, st, grid, cs) : (nv == 2 ? launch_units<NK, 2>(a, st, grid, cs) : launch_units<NK, 4>(a, st, grid, cs));
}

// How many CTAs share a row tile's keys: as many as put two on every SM (a CTA's 8 warps hide half of the latency), each with 4 tiles of keys or more when the block
// table is as long as its sequence.  Up to 8 are a cluster; beyond that several clusters.
struct Plan {
    int64_t tiles;
    int heads, cluster, parts;
};
Plan plan(const b200seq_step& st, const b200seq_attn_desc& d) {
    Plan p;
    const int R = d.H / d.G, Rb = R < ROWS ? R : ROWS, QT = ROWS / Rb;
    p.heads = d.G * ((R + Rb - 1) / Rb);
    p.tiles = st.T == st.B ? st.T : ((int64_t)st.T + QT - 1) / QT + st.B;
    int64_t keys = (int64_t)st.max_blocks * st.block_size;
    if (d.chunk > 0 && d.chunk < keys) keys = d.chunk;
    if (d.window > 0 && (int64_t)d.window + d.keep_first + QT < keys) keys = (int64_t)d.window + d.keep_first + QT;
    int64_t want = 2 * 148 / (p.tiles * p.heads), most = keys / (4 * KT);
    want = want < most ? want : most;
    p.cluster = want >= 8 ? 8 : (want >= 4 ? 4 : (want >= 2 ? 2 : 1));
    p.parts = want >= 16 ? (int)(want / 8 < 16 ? want / 8 : 16) : 1;
    return p;
}

}  // namespace

}  // namespace b200seq

using namespace b200seq;

extern "C" {

size_t b200seq_attn_kv4_scratch_floats(const b200seq_step* st, const b200seq_attn_desc* d) {
    if (!st || !d || st->T < 1 || st->B < 1 || st->block_size < 1 || st->max_blocks < 1 || d->H < 1 || d->G < 1 || d->H % d->G || d->V < 1) return 0;
    const Plan p = plan(*st, *d);
    return p.parts > 1 ? (size_t)st->T * d->H * p.parts * (d->V + 4) : 0;
}

int b200seq_attn_kv4(const float* proj, int64_t ld, const b200seq_step* st, const b200seq_attn_desc* d, const void* kpool, const void* vpool, void* out, int out_dtype,
                     float* scratch, size_t scratch_floats, void* stream) {
    if (int rc = attn_desc_check(d, "attn_kv4")) return rc;
    if (!st || st->T < 0 || st->B < 0 || st->block_size < 1 || st->max_blocks < 0) return fail(B200SEQ_ERR_INVALID_ARG, "attn_kv4: bad step");
    if (!proj || !kpool || !vpool || !out || (st->T > 0 && (!st->tok_pos || !st->ent_start || !st->block_table))) return fail(B200SEQ_ERR_INVALID_ARG, "attn_kv4: bad arguments");
    if (out_dtype != B200SEQ_F32 && out_dtype != B200SEQ_BF16) return fail(B200SEQ_ERR_INVALID_ARG, "attn_kv4: results are f32 or bf16");
    if (d->pool > 0 || d->latent_v || d->krot || d->ctx_rows || d->kv_ld > 0 || (d->kd > 0 && d->kd < d->D))
        return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: a 4-bit cache holds plain keys and values (no pooled blocks, no latents)");
    if (d->D > KV4_MAX_DIM || d->V > KV4_MAX_DIM) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: heads of up to %d values", KV4_MAX_DIM);
    if ((reinterpret_cast<uintptr_t>(kpool) | reinterpret_cast<uintptr_t>(vpool)) & 15) return fail(B200SEQ_ERR_INVALID_ARG, "attn_kv4: pools start on a 16-byte boundary");
    if (st->block_size > 1 << 16) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: pages of up to 65536 tokens");
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
    a.softcap = d->softcap, a.out = out, a.out_dtype = out_dtype, a.err = error_flag_dev();
    Plan p = plan(*st, *d);
    if (p.parts > 1 && (!scratch || scratch_floats < (size_t)st->T * d->H * p.parts * (d->V + 4))) p.parts = 1;
    a.cluster = p.cluster, a.parts = p.parts, a.part = scratch;
    if (p.heads > 65535 || p.tiles * p.parts > 0x7fffffff || d->H > 65535) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: too many heads or tokens");
    const dim3 grid((unsigned)(p.tiles * p.parts), (unsigned)p.heads, (unsigned)p.cluster);
    const int nk = kv4_groups(d->D), nv = kv4_groups(d->V);
    cudaStream_t cs = (cudaStream_t)stream;
    const cudaError_t e = nk == 1 ? launch_values<1>(nv, a, *st, grid, cs) : (nk == 2 ? launch_values<2>(nv, a, *st, grid, cs) : launch_values<4>(nv, a, *st, grid, cs));
    if (e != cudaSuccess) return cuda_status(e, "attn_kv4");
    count_launch();
    if (p.parts > 1) {
        launch_chained(attn4_merge_kernel, dim3(st->T, d->H), d->V <= 64 ? 64 : 128, 0, cs, a);
        SEQ_LAUNCH_CHECK("attn_kv4 merge");
    }
    return 0;
}

}  // extern "C"
