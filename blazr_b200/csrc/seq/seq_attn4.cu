// seq_attn4.cu -- the attend step over KV pages held in 4 bits (seq_kv4.cuh has their layout), in one pass over the keys with a running maximum and sum.
//
// o = sum_j w_j v_j / sum_j w_j,  w_j = exp(z_j - max z),  z_j = scale q . k_j over the keys that a row (token, query head) sees.  With k_j = m + s u (minimum, step and
// code of a group of 32):  q . k_j = sum_groups s (q . u) + m (sum q),  and likewise for v.
//
// A warp has a row tile of up to 8 rows that share a key head and walks over tiles of 16 keys, m16n8k16 products in f16 with f32 sums.  What bounds a decode
// step is the cache's bytes: 8 rows are too few for tcgen05 (128 rows a product, operands through shared memory at four times the cache's width), so the codes are
// expanded in registers, where a key's go straight into an operand:
//   scores  [16 x 8 keys]: the rows are A, q as two f16 numbers (22 bits): rows 0 - 7 the high parts, rows 8 - 15 the low ones, so that both products of a score meet in
//           one thread.  B is a field of the code word ANDed out: the bits 0 .. 15 as an f16 are u 2^-24 or, a field higher, u 2^-20, exactly; q takes the powers in.  s and m
//           enter afterwards in f32.
//   values  [16 x 8 columns]: the weights are A, again in two f16 parts, from the scores' own registers.  B is s u, which is an f16 number; m is summed in f32.
// So nothing is rounded but q and the weights to 22 bits; the rest is f32.
#include "seq_attn4.cuh"
#include "tc_split.cuh"

namespace b200seq {

namespace {

constexpr int KT = 16;        // keys per tile
constexpr int ROWS = 8;       // rows per row tile
constexpr int WARPS = 8;
constexpr int STAGES = 3;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
__device__ __forceinline__ float par_m(uint32_t p) { return __half2float(__ushort_as_half((uint16_t)(p >> 16))); }
__device__ __forceinline__ uint32_t half2_sub_mul(uint32_t x, uint32_t sub, uint32_t mul) {
    const __half2 d = __hmul2_rn(__hsub2_rn(*reinterpret_cast<__half2*>(&x), *reinterpret_cast<__half2*>(&sub)), *reinterpret_cast<__half2*>(&mul));
    return *reinterpret_cast<const uint32_t*>(&d);
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

// a tile of 16 keys from key0 on into shared memory: codes (swizzled), then parameters.  Keys behind `hi` are read from hi's row, or, in whole units, from the
// rest of its page.
template <int NG, bool UNITS>
__device__ __forceinline__ void fetch(uint32_t dst, const uint8_t* pool, const int32_t* bt, int bs, int key0, int hi, int g, int G, int lane) {
    if (UNITS) {
        const int pg = key0 / bs;
        const uint8_t* src = pool + ((int64_t)bt[pg] * G + g) * (int64_t)(bs * NG * 20) + (key0 - pg * bs) * (NG * 20);
#pragma unroll
        for (int i = lane; i < NG * 20; i += 32) copy16(dst + 16 * (i < NG * 16 ? swz(i) : i), src + 16 * i);
    } else {
        for (int i = lane; i < KT * NG * 5; i += 32) {
            const int row = i / (NG * 5), w = i - row * (NG * 5), key = min(key0 + row, hi), pg = key / bs;
            const Kv4Row at = kv4_row(bt[pg], key - pg * bs, bs, g, G, NG);
            if (w < NG * 4) copy4(dst + 16 * swz(row * NG + (w >> 2)) + 4 * (w & 3), pool + at.codes + 4 * w);
            else copy4(dst + NG * 256 + row * NG * 4 + 4 * (w - NG * 4), pool + at.params + 4 * (w - NG * 4));
        }
    }
}

template <int NK, int NV, bool UNITS>
__global__ void __launch_bounds__(WARPS * 32) attn4_kernel(const __grid_constant__ Attn4Args a, const __grid_constant__ b200seq_step st) {
    chain_enter();
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int KB = NK * 320, STAGE = (NK + NV) * 320, MV = 32 * NV + 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int D = a.D, V = a.V, R = a.H / a.G, bs = st.block_size;
    int e, t0, nq;
    if (st.T == st.B) e = t0 = blockIdx.x, nq = 1;
    else if (!attn_find_tile(st, blockIdx.x, a.QT, e, t0, nq)) return;
    const int g = blockIdx.y / a.HB, hb = blockIdx.y - g * a.HB, h0 = g * R + hb * a.Rb, nh = min(a.Rb, R - hb * a.Rb);
    const int p0 = st.tok_pos[t0], hi = p0 + nq - 1;
    const int32_t* bt = st.block_table + (int64_t)e * st.max_blocks;
    if (p0 < 0 || hi / bs >= st.max_blocks) {
        if (threadIdx.x == 0) atomicOr(a.err, 1);
        return;
    }
    const KeySpan<KT> span(a, p0, hi);
    // this thread's row: q as A fragments (eight neighbouring values of every group), its factor and what it sees
    const int tq = r / a.Rb, hr = r - tq * a.Rb;
    const bool live = tq < nq && hr < nh;
    const RowSpan rs(a, p0 + (live ? tq : 0));
    uint32_t qa[NK][2][4];
    float qs[NK], zf;
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
        // times a power of two that puts the largest into [2^10, 2^11); a row of zeros, denormals or infinities as it is
        const int ex = (int)(__float_as_uint(mx) >> 23);
        const bool norm = ex >= 20 && ex < 255;
        // (with the sign of the factor: what follows is scaled by its magnitude)
        float factor = a.scale;
        if (live && a.head_scale) factor *= a.head_scale[h0 + hr];
        const float up = copysignf(norm ? __uint_as_float((uint32_t)(254 - ex + 10) << 23) : 1.f, factor), down = norm ? __uint_as_float((uint32_t)(ex - 10) << 23) : 1.f;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[k][i] *= up, sum += x[k][i];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1), sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            qs[k] = sum * 0x1p-24f;
#pragma unroll
            for (int s = 0; s < 2; ++s) {   // fields 0 and 4 (2 and 6) of a word, then 1 and 5 (3 and 7), which stand four bits higher
                split16(x[k][2 * s], x[k][2 * s + 4], qa[k][s][0], qa[k][s][1]);
                split16(x[k][2 * s + 1] * 0.0625f, x[k][2 * s + 5] * 0.0625f, qa[k][s][2], qa[k][s][3]);
            }
        }
        zf = fmaxf(fabsf(factor) * (a.softcap > 0.f ? 1.f : LOG2E), 1e-37f) * down * 0x1p24f;
    }
    float mx = -INFINITY, l = 0.f, om[NV], o[NV * 4][4];
#pragma unroll
    for (int k = 0; k < NV; ++k) om[k] = 0.f;
#pragma unroll
    for (int k = 0; k < NV * 4; ++k) o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;

    const uint32_t ring = tcpair::sa(smem) + warp * (STAGES * STAGE);
    const int nt = span.total > warp ? (span.total - warp + WARPS - 1) / WARPS : 0;
    auto issue = [&](int i) {
        if (i < nt) {
            const int key0 = span.key0(warp + i * WARPS);
            const uint32_t dst = ring + (i % STAGES) * STAGE;
            fetch<NK, UNITS>(dst, a.kpool, bt, bs, key0, hi, g, a.G, lane);
            fetch<NV, UNITS>(dst + KB, a.vpool, bt, bs, key0, hi, g / a.vdiv, a.G / a.vdiv, lane);
        }
        copies_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i);
#pragma unroll 1
    for (int i = 0; i < nt; ++i) {
        issue(i + STAGES - 1);
        copies_wait<STAGES - 1>();
        __syncwarp();
        const uint32_t ks = ring + (i % STAGES) * STAGE, vs = ks + KB;
        const int key0 = span.key0(warp + i * WARPS);
        // ---- scores of keys key0 + {2c, 2c + 1, 8 + 2c, 9 + 2c} ----
        float z[4];
        {
            uint32_t kw[2][NK], kp[4][NK];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int row = r + 8 * n;
                lds<NK>(ks + (NK == 4 ? 16 * swz(row * 4 + c) : (NK == 2 ? 16 * swz(row * 2 + (c >> 1)) + 8 * (c & 1) : 16 * swz(row) + 4 * c)), kw[n]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) lds<NK>(ks + NK * 256 + (2 * c + (j & 1) + 8 * (j >> 1)) * NK * 4, kp[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j) z[j] = 0.f;
#pragma unroll
            for (int k = 0; k < NK; ++k) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
                    const uint32_t w = kw[n][k], w8 = w >> 8;
                    mma16816(acc, qa[k][0], w & 0x000F000Fu, w & 0x00F000F0u);
                    mma16816(acc, qa[k][1], w8 & 0x000F000Fu, w8 & 0x00F000F0u);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t p = kp[2 * n + j][k];
                        z[2 * n + j] = fmaf(acc[j] + acc[2 + j], par_s(p), fmaf(par_m(p), qs[k], z[2 * n + j]));
                    }
                }
            }
        }
        float tm = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (a.softcap > 0.f) z[j] = a.softcap * LOG2E * tanhf(z[j] * zf / a.softcap);
            if (!rs.sees(key0 + 2 * c + (j & 1) + 8 * (j >> 1))) z[j] = -INFINITY;
            tm = fmaxf(tm, a.softcap > 0.f ? z[j] : z[j] * zf);
        }
        tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 1)), tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 2));
        const float mn = fmaxf(mx, tm), off = mn == -INFINITY ? 0.f : mn;
        if (__any_sync(0xffffffffu, mn > mx)) {
            const float corr = tcsplit::ex2(mx - off);   // 0 at the first key a row sees
            l *= corr;
#pragma unroll
            for (int k = 0; k < NV; ++k) om[k] *= corr;
#pragma unroll
            for (int k = 0; k < NV * 4; ++k) o[k][0] *= corr, o[k][1] *= corr, o[k][2] *= corr, o[k][3] *= corr;
        }
        mx = mn;
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = tcsplit::ex2(a.softcap > 0.f ? z[j] - off : fmaf(z[j], zf, -off)), l += p[j];
        uint32_t pa[4];
        split16(p[0], p[1], pa[0], pa[1]);
        split16(p[2], p[3], pa[2], pa[3]);
        // ---- values ----
        {
            uint32_t vp[4][NV], vw[4][(NV + 1) / 2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = 2 * c + (j & 1) + 8 * (j >> 1);
                lds<NV>(vs + NV * 256 + row * NV * 4, vp[j]);
                if (NV == 4) lds<(NV + 1) / 2>(vs + 16 * swz(row * 4 + (r >> 1)) + 8 * (r & 1), vw[j]);
                else if (NV == 2) lds<(NV + 1) / 2>(vs + 16 * swz(row * 2 + (r >> 2)) + 4 * (r & 3), vw[j]);
                else vw[j][0] = lds16(vs + 16 * swz(row) + 2 * r);
                if (key0 + row > hi) {   // whatever lies behind the last key
#pragma unroll
                    for (int k = 0; k < NV; ++k) vp[j][k] = 0;
                }
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint32_t s0 = __byte_perm(vp[0][k], vp[1][k], 0x5410), s1 = __byte_perm(vp[2][k], vp[3][k], 0x5410);
                const int sel = (k & 1) ? 0x7632 : 0x5410;
                const uint32_t x0 = __byte_perm(vw[0][k >> 1], vw[1][k >> 1], sel), x1 = __byte_perm(vw[2][k >> 1], vw[3][k >> 1], sel);
#pragma unroll
                for (int j = 0; j < 4; ++j) om[k] = fmaf(p[j], par_m(vp[j][k]), om[k]);
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    const uint32_t b0 = half2_sub_mul(((x0 >> (4 * i4)) & 0x000F000Fu) | 0x64006400u, 0x64006400u, s0);
                    const uint32_t b1 = half2_sub_mul(((x1 >> (4 * i4)) & 0x000F000Fu) | 0x64006400u, 0x64006400u, s1);
                    mma16816(o[4 * k + i4], pa, b0, b1);
                }
            }
        }
        __syncwarp();   // the stage is refilled next
    }
    copies_wait<0>();
    // ---- the warps' parts: [row][max, sum, values] in shared memory, over the ring ----
    l += __shfl_xor_sync(0xffffffffu, l, 1), l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
    for (int k = 0; k < NV; ++k) om[k] += __shfl_xor_sync(0xffffffffu, om[k], 1), om[k] += __shfl_xor_sync(0xffffffffu, om[k], 2);
    __syncthreads();
    float* part = reinterpret_cast<float*>(smem) + (warp * ROWS + r) * MV;
    if (c == 0) part[0] = mx, part[1] = l;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
            for (int j = 0; j < 2; ++j) part[4 + 32 * k + 8 * c + 4 * j + i4] = o[4 * k + i4][j] + o[4 * k + i4][2 + j] + om[k];
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(smem);
    for (int i = threadIdx.x; i < nq * nh * V; i += blockDim.x) {
        const int m = i / V, col = i - m * V, tq_ = m / nh, hr_ = m - tq_ * nh, t = t0 + tq_, h = h0 + hr_;
        const float* pr = all + (tq_ * a.Rb + hr_) * MV;
        const float sk = a.sink ? a.sink[h] * LOG2E : -INFINITY;
        float M = sk;
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, pr[w * ROWS * MV]);
        float L = a.sink ? tcsplit::ex2(sk - M) : 0.f, acc = 0.f;
        for (int w = 0; w < WARPS; ++w) {
            if (pr[w * ROWS * MV + 1] == 0.f) continue;   // this warp had no key that the row sees
            const float f = tcsplit::ex2(pr[w * ROWS * MV] - M);
            L = fmaf(pr[w * ROWS * MV + 1], f, L), acc = fmaf(pr[w * ROWS * MV + 4 + col], f, acc);
        }
        float gate = 1.f;
        if (a.gated) gate = sigmoidf_acc(a.gate[(int64_t)t * a.gld + (a.gate_elem ? (int64_t)h * V + col : h)]);
        store_act(a.out, a.out_dtype, ((int64_t)t * a.H + h) * V + col, acc / L * gate);
    }
}

template <int NK, int NV, bool UNITS>
cudaError_t launch(const Attn4Args& a, const b200seq_step& st, dim3 grid, cudaStream_t cs) {
    constexpr int ring = WARPS * STAGES * (NK + NV) * 320, parts = WARPS * ROWS * (32 * NV + 4) * 4, smem = ring > parts ? ring : parts;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(attn4_kernel<NK, NV, UNITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
    }
    launch_chained(attn4_kernel<NK, NV, UNITS>, grid, WARPS * 32, smem, cs, a, st);
    return cudaGetLastError();
}
template <int NK, int NV>
cudaError_t launch_units(const Attn4Args& a, const b200seq_step& st, dim3 grid, cudaStream_t cs) {
    return st.block_size % 16 == 0 ? launch<NK, NV, true>(a, st, grid, cs) : launch<NK, NV, false>(a, st, grid, cs);
}
template <int NK>
cudaError_t launch_values(int nv, const Attn4Args& a, const b200seq_step& st, dim3 grid, cudaStream_t cs) {
    return nv == 1 ? launch_units<NK, 1>(a, st, grid, cs) : (nv == 2 ? launch_units<NK, 2>(a, st, grid, cs) : launch_units<NK, 4>(a, st, grid, cs));
}

}  // namespace

}  // namespace b200seq

using namespace b200seq;

extern "C" {

int b200seq_attn_kv4(const float* proj, int64_t ld, const b200seq_step* st, const b200seq_attn_desc* d, const void* kpool, const void* vpool, void* out, int out_dtype,
                     void* stream) {
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
    const int64_t tiles = st->T == st->B ? st->T : (st->T + a.QT - 1) / a.QT + st->B, heads = (int64_t)d->G * a.HB;
    if (heads > 65535 || tiles > 0x7fffffff) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_kv4: too many heads or tokens");
    const dim3 grid((unsigned)tiles, (unsigned)heads);
    const int nk = kv4_groups(d->D), nv = kv4_groups(d->V);
    const cudaError_t e = nk == 1 ? launch_values<1>(nv, a, *st, grid, (cudaStream_t)stream)
                                  : (nk == 2 ? launch_values<2>(nv, a, *st, grid, (cudaStream_t)stream) : launch_values<4>(nv, a, *st, grid, (cudaStream_t)stream));
    if (e != cudaSuccess) return cuda_status(e, "attn_kv4");
    count_launch();
    return 0;
}

}  // extern "C"
