// seq_kv4.cu -- keys and values into and out of a cache held in 4 bits (layout and rounding: seq_kv4.cuh).
#include "seq_kv4.cuh"

namespace b200seq {

namespace {

struct Kv4Rows {
    const void *k, *v;
    int64_t ldk, ldv;
    uint8_t *kpool, *vpool;
    int G, D, Gv, V, vec;
};

// position of a token in its sequence's pages; negative (and the error flag) outside the block table or where the table has no page
__device__ __forceinline__ int kv4_page(const b200seq_step& st, int t, int& o, int* err) {
    const int pos = st.tok_pos[t], b = pos / st.block_size;
    o = pos - b * st.block_size;
    if (pos < 0 || b >= st.max_blocks) {
        atomicOr(err, 1);
        return -1;
    }
    const int page = st.block_table[(int64_t)st.tok_ent[t] * st.max_blocks + b];
    if (page < 0) atomicOr(err, 1);
    return page;
}

// A lane's eight codes and its group's parameters into a row.  Lanes of neighbouring groups change halves, so that value codes are stored as 32-bit words too.
// All lanes of the warp take part; those with `in` store.
__device__ __forceinline__ void kv4_put(uint8_t* pool, const Kv4Row& at, bool key, int hl, int NG, uint32_t w, uint32_t param, bool in) {
    const bool second = hl & 4;                    // an odd group
    const uint32_t other = __shfl_xor_sync(0xffffffffu, second ? w & 0xFFFFu : w >> 16, 4);
    if (!in || hl >= 4 * NG) return;
    uint8_t* p = pool + at.codes;
    if (key) {
        *reinterpret_cast<uint32_t*>(p + kv4_key_place(hl, NG)) = w;
    } else if (NG == 1) {
        *reinterpret_cast<uint16_t*>(p + kv4_value_place(hl, NG)) = (uint16_t)w;
        *reinterpret_cast<uint16_t*>(p + kv4_value_place(hl, NG) + 2 * NG) = (uint16_t)(w >> 16);
    } else {                                       // the even group of a pair stores the first words of both, the odd one the second
        *reinterpret_cast<uint32_t*>(p + kv4_value_place(hl & ~4, NG) + (second ? 2 * NG : 0)) = second ? other | (w & 0xFFFF0000u) : (w & 0xFFFFu) | (other << 16);
    }
    if ((hl & 3) == 0) *reinterpret_cast<uint32_t*>(pool + at.params + hl) = param;
}

// A block has a token; LPR lanes (4 for every group of the wider of key and value heads) have a row of it at a time.  WHOLE: keys and values of as many groups,
// rows of whole 16-byte pieces, of bf16 values or not.  Bounded by instructions: about 300 a pair of rows (4094 tokens of 16 rows of 128 bf16 values, stored and loaded: 22.4 us, 26.0 with the rows asked for behind their page).
template <int LPR, bool WHOLE, bool BF16>
__global__ void __launch_bounds__(256) kv4_store_kernel(const Kv4Rows a, const b200seq_step st, int* err) {
    chain_enter();
    const int hl = threadIdx.x & (LPR - 1), heads = a.G + a.Gv, t = blockIdx.x;
    float x[8];
    auto fetch = [&](int u) {
        const bool key = u < a.G;
        const int g = key ? u : u - a.G, D = key ? a.D : a.V, n = u < heads ? min(max(D - 8 * hl, 0), 8) : 0;
        const int64_t src = (int64_t)t * (key ? a.ldk : a.ldv) + (g * D + 8 * hl);
        const void* p = key ? a.k : a.v;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
        if (BF16) {
            const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p) + src;
            if (WHOLE) {
                const uint4 w = n ? *reinterpret_cast<const uint4*>(q) : make_uint4(0, 0, 0, 0);
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) x[2 * j] = __uint_as_float(ws[j] << 16), x[2 * j + 1] = __uint_as_float(ws[j] & 0xFFFF0000u);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n) x[j] = __bfloat162float(q[j]);
            }
        } else {
            const float* q = reinterpret_cast<const float*>(p) + src;
            if (WHOLE) {
                if (n) {
                    const float4 v = ld4(q), w = ld4(q + 4);
                    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w, x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n) x[j] = q[j];
            }
        }
    };
    fetch((int)threadIdx.x / LPR);                 // (on its way while the page is looked up)
    int o;
    const int page = kv4_page(st, t, o, err);
    if (page < 0) return;
    bool odd = false;
    for (int u0 = (threadIdx.x & ~31) / LPR; u0 < heads; u0 += blockDim.x / LPR) {
        const int u = u0 + (threadIdx.x & 31) / LPR;
        const bool in = u < heads, key = u < a.G;
        const int g = key ? u : u - a.G, D = key ? a.D : a.V, NG = WHOLE ? LPR / 4 : kv4_groups(D), n = in ? min(max(D - 8 * hl, 0), 8) : 0;
        uint32_t param;
        const uint32_t w = kv4_quantise(x, n, param, odd);
        kv4_put(key ? a.kpool : a.vpool, kv4_row(page, o, st.block_size, in ? g : 0, key ? a.G : a.Gv, NG), key, hl, NG, w, param, in);
        if (u0 + (int)blockDim.x / LPR < heads) fetch(u + (int)blockDim.x / LPR);
    }
    if (odd) atomicOr(err, KV4_ERR_RANGE);
}
template <bool WHOLE, bool BF16>
auto store_kernel(int lpr) {
    return lpr == 4 ? kv4_store_kernel<4, WHOLE, BF16> : (lpr == 8 ? kv4_store_kernel<8, WHOLE, BF16> : kv4_store_kernel<16, WHOLE, BF16>);
}

// The same rows back, as the values they stand for.  A block has TOK tokens: two where half the GPU's threads have work (4094 tokens of 16 rows of 128: 22.4
// us for storing and loading with two, 23.9 with one; 300 tokens 4.9 and 4.6).
template <int LPR, bool WHOLE, int TOK>
__global__ void __launch_bounds__(256) kv4_load_kernel(const Kv4Rows a, float* __restrict__ ko, float* __restrict__ vo, const b200seq_step st, int* err) {
    chain_enter();
    const int hl = threadIdx.x & (LPR - 1), heads = a.G + a.Gv, t0 = blockIdx.x * TOK;
    int o[TOK], page[TOK];
#pragma unroll
    for (int k = 0; k < TOK; ++k) page[k] = t0 + k < st.T ? kv4_page(st, t0 + k, o[k], err) : -1;
    for (int u = threadIdx.x / LPR; u < heads; u += blockDim.x / LPR) {
        const bool key = u < a.G;
        const int g = key ? u : u - a.G, D = key ? a.D : a.V, NG = WHOLE ? LPR / 4 : kv4_groups(D), n = min(max(D - 8 * hl, 0), 8);
        if (n == 0) continue;
        const uint8_t* pool = key ? a.kpool : a.vpool;
        uint32_t w[TOK], pr[TOK];
#pragma unroll
        for (int k = 0; k < TOK; ++k) {
            w[k] = pr[k] = 0;
            if (page[k] < 0) continue;
            const Kv4Row at = kv4_row(page[k], o[k], st.block_size, g, key ? a.G : a.Gv, NG);
            if (key) w[k] = *reinterpret_cast<const uint32_t*>(pool + at.codes + kv4_key_place(hl, NG));
            else w[k] = *reinterpret_cast<const uint16_t*>(pool + at.codes + kv4_value_place(hl, NG)) | ((uint32_t)*reinterpret_cast<const uint16_t*>(pool + at.codes + kv4_value_place(hl, NG) + 2 * NG) << 16);
            pr[k] = *reinterpret_cast<const uint32_t*>(pool + at.params + (hl & ~3));
        }
        float* dst = (key ? ko + (int64_t)t0 * a.ldk : vo + (int64_t)t0 * a.ldv) + g * D + 8 * hl;
#pragma unroll
        for (int k = 0; k < TOK; ++k, dst += key ? a.ldk : a.ldv) {
            if (page[k] < 0) continue;
            const float s = __half2float(__ushort_as_half((uint16_t)pr[k])), m = __half2float(__ushort_as_half((uint16_t)(pr[k] >> 16)));
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = fmaf(s, __uint_as_float(((w[k] >> (4 * j)) & 15u) | 0x4B000000u) - 8388608.f, m);   // (2^23 + code)
            if (WHOLE) {
                *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n) dst[j] = x[j];
            }
        }
    }
}
template <bool WHOLE, int TOK>
auto load_kernel(int lpr) {
    return lpr == 4 ? kv4_load_kernel<4, WHOLE, TOK> : (lpr == 8 ? kv4_load_kernel<8, WHOLE, TOK> : kv4_load_kernel<16, WHOLE, TOK>);
}

// b200seq_attn_prep_ex over 4-bit pages, for rows of whole 16-byte pieces (every head size, rotation and column that is a multiple of 8; norms over single heads).
// LPR lanes have a head's row (4 for every group of 32), eight neighbouring values in a lane's registers; the rotation's other half comes from another lane.
// A token's rows are split over `split` blocks of 128 threads.  Bounded by a chain of loads for single tokens (position, frequencies, then sines); for prompts
// by that chain and by instructions (2048 tokens: issue slots 56 % active, a warp waits 5 of 12 cycles for loads from memory, DRAM 20 %).  us with rotation of halves and norms, rows as here / a warp to a head through shared memory (32 query heads of 8 key heads of 128):
//   1 token  2.9 / 8.7      32 tokens  3.3 / 9.5      512  8.9 / 14.1      2048  26.3 / 49.9  (bytes alone: 12.8)
template <int LPR>
__global__ void __launch_bounds__(128) kv4_prep_rows_kernel(float* proj, int64_t ld, const b200seq_step st, const b200seq_attn_desc a, uint8_t* kpool, uint8_t* vpool,
                                                            int split, int* err) {
    chain_enter();
    extern __shared__ __align__(16) float rot_sm[];   // cos | sin
    constexpr int ROWS = 128 / LPR;
    const int t = blockIdx.x / split, part = blockIdx.x - t * split, lane = threadIdx.x & 31, hl = threadIdx.x & (LPR - 1);
    const int pos = st.tok_pos[t];
    const int H = a.H, G = a.G, Gv = a.vg > 0 ? a.vg : G, np = a.rot_dims >> 1, nu = a.kv_shared ? H : H + G + Gv;
    int o = 0;
    const int page = a.kv_shared ? -1 : kv4_page(st, t, o, err);
    float* base = proj + (int64_t)t * ld;
    bool odd = false, first = true;
    for (int u0 = part * ROWS; u0 < nu; u0 += split * ROWS) {
        const int u = u0 + (int)threadIdx.x / LPR;
        const bool in = u < nu, isq = u < H, isk = !isq && u < H + G, turned = in && (isq || isk);
        const int hh = isq ? u : (isk ? u - H : u - H - G), size = isq || isk ? a.D : a.V, n = in && 8 * hl < size ? 8 : 0;
        const int col = (isq ? a.q_col : (isk ? a.k_col : a.v_col)) + hh * size + 8 * hl;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
        if (n) {
            const float4 v = ld4(base + col), w = ld4(base + col + 4);
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w, x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
            if (a.in_bias) {
                const float4 b = ld4(a.in_bias + col), c = ld4(a.in_bias + col + 4);
                x[0] += b.x, x[1] += b.y, x[2] += b.z, x[3] += b.w, x[4] += c.x, x[5] += c.y, x[6] += c.z, x[7] += c.w;
            }
        }
        if (first) {
            for (int i = threadIdx.x; i < np; i += 128) {
                float sn, cs;
                sincosf((float)(a.rot_pos ? a.rot_pos[t] : pos) * a.rot_freq[i], &sn, &cs);
                rot_sm[i] = cs * a.rot_scale, rot_sm[np + i] = sn * a.rot_scale;
            }
            __syncthreads();
            first = false;
        }
        if (a.qk_eps >= 0.f) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
            for (int m = 1; m < LPR; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
            if (turned && n) {
                const float* w = isq ? a.q_norm_w : a.k_norm_w;
                const float rinv = 1.0f / sqrtf(ss / (float)a.D + a.qk_eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= rinv;
                if (w) {
                    const float4 b = ld4(w + 8 * hl), c = ld4(w + 8 * hl + 4);
                    x[0] *= b.x, x[1] *= b.y, x[2] *= b.z, x[3] *= b.w, x[4] *= c.x, x[5] *= c.y, x[6] *= c.z, x[7] *= c.w;
                }
            }
        }
        if (np > 0 && a.rot_half) {
            const bool lower = 8 * hl < np, turns = turned && 8 * hl < 2 * np;
            const int from = 8 * hl >= 2 * np ? lane : (lower ? lane + (np >> 3) : lane - (np >> 3)), i = lower ? 8 * hl : 8 * hl - np;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float other = __shfl_sync(0xffffffffu, x[j], from);
                if (turns) x[j] = fmaf(x[j], rot_sm[i + j], (lower ? -other : other) * rot_sm[np + i + j]);
            }
        } else if (turned) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = 4 * hl + j;
                if (i >= np) continue;
                const float e = x[2 * j], f = x[2 * j + 1], cs = rot_sm[i], sn = rot_sm[np + i];
                x[2 * j] = fmaf(e, cs, -f * sn), x[2 * j + 1] = fmaf(f, cs, e * sn);
            }
        }
        if (isq) {
            if (n) {
                *reinterpret_cast<float4*>(base + col) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4*>(base + col + 4) = make_float4(x[4], x[5], x[6], x[7]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.f;   // (a query is none of the values that are held)
        }
        if (page >= 0 && __any_sync(0xffffffffu, in && !isq)) {
            const int NG = kv4_groups(size);
            uint32_t param;
            const uint32_t w = kv4_quantise(x, isq ? 0 : n, param, odd);
            kv4_put(isk ? kpool : vpool, kv4_row(page, o, st.block_size, in && !isq ? hh : 0, isk ? G : Gv, NG), isk, hl, NG, w, param, in && !isq);
        }
    }
    if (odd) atomicOr(err, KV4_ERR_RANGE);
}

// The same for every other row: grid (T), 256 threads, a warp per head unit; the unit's values are staged in the warp's slice of shared memory, biased,
// normed, turned, and written back (queries) or quantised into the token's row.  Shared memory: rot_dims floats (cos | sin) + 8 * Dmax + 40.
__global__ void kv4_prep_kernel(float* __restrict__ proj, int64_t ld, const b200seq_step st, const b200seq_attn_desc a, uint8_t* __restrict__ kpool,
                                uint8_t* __restrict__ vpool, int Dmax, int* err) {
    chain_enter();
    extern __shared__ float gsm[];
    float* rot_sm = gsm;
    float* stage = gsm + a.rot_dims;
    float* red = stage + 8 * Dmax;
    const int t = blockIdx.x, lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
    const int pos = st.tok_pos[t];
    const int H = a.H, G = a.G, D = a.D, V = a.V, Gv = a.vg > 0 ? a.vg : G, np = a.rot_dims >> 1;
    int o = 0;
    const int page = a.kv_shared ? -1 : kv4_page(st, t, o, err);
    float* base = proj + (int64_t)t * ld;
    for (int i = threadIdx.x; i < np; i += blockDim.x) {
        float sn, cs;
        sincosf((float)(a.rot_pos ? a.rot_pos[t] : pos) * a.rot_freq[i], &sn, &cs);
        rot_sm[i] = cs * a.rot_scale, rot_sm[np + i] = sn * a.rot_scale;
    }
    auto biased = [&](int col) { return base[col] + (a.in_bias ? a.in_bias[col] : 0.f); };
    float rq = 1.f, rk = 1.f;
    if (a.norm_full && a.qk_eps >= 0.f) {
        float sq = 0.f, sk = 0.f;
        for (int i = threadIdx.x; i < H * D; i += blockDim.x) sq = fmaf(biased(a.q_col + i), biased(a.q_col + i), sq);
        rq = 1.0f / sqrtf(block_sum(sq, red) / (float)(H * D) + a.qk_eps);
        if (!a.kv_shared) {
            for (int i = threadIdx.x; i < G * D; i += blockDim.x) sk = fmaf(biased(a.k_col + i), biased(a.k_col + i), sk);
            rk = 1.0f / sqrtf(block_sum(sk, red) / (float)(G * D) + a.qk_eps);
        }
    }
    __syncthreads();   // rot_sm
    float* hs = stage + wid * Dmax;
    bool odd = false;
    const int nu = a.kv_shared ? H : H + G + Gv;
    for (int u = wid; u < nu; u += nw) {
        const bool isq = u < H, isk = !isq && u < H + G;
        const int hh = isq ? u : (isk ? u - H : u - H - G), size = isq || isk ? D : V;
        const int col = (isq ? a.q_col : (isk ? a.k_col : a.v_col)) + hh * size;
        float ss = 0.f;
        for (int d = lane; d < size; d += 32) {
            const float v = biased(col + d);
            hs[d] = v;
            ss = fmaf(v, v, ss);
        }
        if (isq || isk) {
            const float* w = isq ? a.q_norm_w : a.k_norm_w;
            if (a.qk_eps >= 0.f) {
                const float rinv = a.norm_full ? (isq ? rq : rk) : 1.0f / sqrtf(warp_sum(ss) / (float)D + a.qk_eps);
                for (int d = lane; d < D; d += 32) hs[d] = hs[d] * rinv * (w ? w[a.norm_full ? hh * D + d : d] : 1.f);
            }
            __syncwarp();
            for (int i = lane; i < np; i += 32) {   // a lane turns whole pairs
                const int d0 = a.rot_half ? i : 2 * i, d1 = a.rot_half ? i + np : 2 * i + 1;
                const float x = hs[d0], y = hs[d1], cs = rot_sm[i], sn = rot_sm[np + i];
                hs[d0] = fmaf(x, cs, -y * sn), hs[d1] = fmaf(y, cs, x * sn);
            }
        }
        __syncwarp();
        if (isq) {
            for (int d = lane; d < D; d += 32) base[col + d] = hs[d];
        } else if (page >= 0) {
            const int n = min(max(size - 8 * lane, 0), 8), NG = kv4_groups(size);
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = i < n ? hs[8 * lane + i] : 0.f;
            uint32_t param;
            const uint32_t w = kv4_quantise(x, n, param, odd);
            kv4_put(isk ? kpool : vpool, kv4_row(page, o, st.block_size, hh, isk ? G : Gv, NG), isk, lane, NG, w, param, true);
        }
        __syncwarp();   // hs is used again by the warp's next unit
    }
    if (odd) atomicOr(err, KV4_ERR_RANGE);
}

int step_check(const b200seq_step* st, const char* what) {
    if (!st || st->T < 0 || st->B < 0 || st->block_size < 1 || st->max_blocks < 0) return fail(B200SEQ_ERR_INVALID_ARG, "%s: bad step", what);
    if (st->T > 0 && (!st->tok_ent || !st->tok_pos || !st->block_table)) return fail(B200SEQ_ERR_INVALID_ARG, "%s: the step lacks its arrays", what);
    if (st->block_size > 1 << 16) return fail(B200SEQ_ERR_UNSUPPORTED, "%s: pages of up to 65536 tokens", what);
    return 0;
}

int rows_check(const b200seq_step* st, const void* k, const void* v, int64_t ldk, int64_t ldv, int G, int D, int Gv, int V, const void* kpool, const void* vpool, const char* what) {
    if (int rc = step_check(st, what)) return rc;
    if (G < 1 || Gv < 1 || D < 1 || V < 1 || !kpool || !vpool || (st->T > 0 && (!k || !v))) return fail(B200SEQ_ERR_INVALID_ARG, "%s: bad sizes or null arrays", what);
    if (D > KV4_MAX_DIM || V > KV4_MAX_DIM) return fail(B200SEQ_ERR_UNSUPPORTED, "%s: heads of up to %d values", what, KV4_MAX_DIM);
    if (st->T > 1 && (ldk < (int64_t)G * D || ldv < (int64_t)Gv * V)) return fail(B200SEQ_ERR_INVALID_ARG, "%s: row strides below a row's length", what);
    if ((reinterpret_cast<uintptr_t>(kpool) | reinterpret_cast<uintptr_t>(vpool)) & 15) return fail(B200SEQ_ERR_INVALID_ARG, "%s: pools start on a 16-byte boundary", what);
    if (!kv4_pages_fit(st->block_size, G, D) || !kv4_pages_fit(st->block_size, Gv, V)) return fail(B200SEQ_ERR_UNSUPPORTED, "%s: pages of up to 2 GiB", what);
    if (((int64_t)G + Gv) * KV4_MAX_DIM > 0x7fffffff) return fail(B200SEQ_ERR_UNSUPPORTED, "%s: too many heads", what);
    return 0;
}

// threads of a block: a token's rows at once, 256 at most
int row_threads(int heads, int lpr) {
    const int n = (heads * lpr + 31) / 32 * 32;
    return n < 256 ? n : 256;
}
// rows whose lanes' eight values are whole 16-byte pieces (align: elements of one)
bool row_pieces(const void* k, const void* v, int64_t ldk, int64_t ldv, int D, int V, int align) {
    return ((D | V) & 7) == 0 && ((ldk | ldv) & (align - 1)) == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
}

}  // namespace

}  // namespace b200seq

using namespace b200seq;

extern "C" {

int64_t b200seq_kv4_page_bytes(int block_size, int G, int D) {
    if (block_size < 1 || G < 1 || D < 1 || D > KV4_MAX_DIM) return 0;
    return (int64_t)block_size * G * kv4_groups(D) * 20;
}

int b200seq_kv4_store(const void* k, int64_t ldk, const void* v, int64_t ldv, int in_dtype, const b200seq_step* st, int G, int D, int Gv, int V, void* kpool, void* vpool,
                      void* stream) {
    if (in_dtype != B200SEQ_F32 && in_dtype != B200SEQ_BF16) return fail(B200SEQ_ERR_INVALID_ARG, "kv4_store: rows are f32 or bf16");
    if (int rc = rows_check(st, k, v, ldk, ldv, G, D, Gv, V, kpool, vpool, "kv4_store")) return rc;
    if (st->T == 0) return 0;
    const bool bf16 = in_dtype == B200SEQ_BF16;
    const Kv4Rows a{k, v, ldk, ldv, (uint8_t*)kpool, (uint8_t*)vpool, G, D, Gv, V, row_pieces(k, v, ldk, ldv, D, V, bf16 ? 8 : 4)};
    const int lpr = 4 * kv4_groups(D > V ? D : V);
    const bool whole = a.vec && kv4_groups(D) == kv4_groups(V);
    launch_chained(whole ? (bf16 ? store_kernel<true, true>(lpr) : store_kernel<true, false>(lpr)) : (bf16 ? store_kernel<false, true>(lpr) : store_kernel<false, false>(lpr)), st->T, row_threads(G + Gv, lpr), 0, (cudaStream_t)stream, a, *st, error_flag_dev());
    SEQ_LAUNCH_CHECK("kv4_store");
    return 0;
}

int b200seq_kv4_load(const void* kpool, const void* vpool, const b200seq_step* st, int G, int D, int Gv, int V, float* k, int64_t ldk, float* v, int64_t ldv, void* stream) {
    if (int rc = rows_check(st, k, v, ldk, ldv, G, D, Gv, V, kpool, vpool, "kv4_load")) return rc;
    if (st->T == 0) return 0;
    const Kv4Rows a{nullptr, nullptr, ldk, ldv, (uint8_t*)kpool, (uint8_t*)vpool, G, D, Gv, V, row_pieces(k, v, ldk, ldv, D, V, 4)};
    const int lpr = 4 * kv4_groups(D > V ? D : V);
    const bool whole = a.vec && kv4_groups(D) == kv4_groups(V);
    const int tok = whole && (int64_t)st->T * (G + Gv) * lpr >= 148 * 1024 ? 2 : 1;
    launch_chained(whole ? (tok == 2 ? load_kernel<true, 2>(lpr) : load_kernel<true, 1>(lpr)) : load_kernel<false, 1>(lpr), (st->T + tok - 1) / tok, row_threads(G + Gv, lpr), 0, (cudaStream_t)stream, a, k, v, *st, error_flag_dev());
    SEQ_LAUNCH_CHECK("kv4_load");
    return 0;
}

int b200seq_attn_prep_kv4(float* proj, int64_t ld, const b200seq_step* st, const b200seq_attn_desc* d, void* kpool, void* vpool, void* stream) {
    if (int rc = step_check(st, "attn_prep_kv4")) return rc;
    if (int rc = attn_desc_check(d, "attn_prep_kv4")) return rc;
    if (!proj || ((!kpool || !vpool) && !d->kv_shared)) return fail(B200SEQ_ERR_INVALID_ARG, "attn_prep_kv4: bad arguments");
    if (d->pool > 0 || d->latent_v || d->krot || d->ctx_rows) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_prep_kv4: a 4-bit cache holds plain keys and values (no pooled blocks, no latents)");
    if (d->D > KV4_MAX_DIM || d->V > KV4_MAX_DIM) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_prep_kv4: heads of up to %d values", KV4_MAX_DIM);
    if ((reinterpret_cast<uintptr_t>(kpool) | reinterpret_cast<uintptr_t>(vpool)) & 15) return fail(B200SEQ_ERR_INVALID_ARG, "attn_prep_kv4: pools start on a 16-byte boundary");
    if (!kv4_pages_fit(st->block_size, d->G, d->D) || !kv4_pages_fit(st->block_size, d->vg > 0 ? d->vg : d->G, d->V)) return fail(B200SEQ_ERR_UNSUPPORTED, "attn_prep_kv4: pages of up to 2 GiB");
    if (st->T == 0) return 0;
    const int Dmax = d->D > d->V ? d->D : d->V;
    const size_t smem = (size_t)(d->rot_dims + 8 * Dmax + 40) * sizeof(float);
    const int heads = d->H + (d->kv_shared ? 0 : d->G + (d->vg > 0 ? d->vg : d->G)), lpr = 4 * kv4_groups(Dmax), np = d->rot_dims / 2;
    const uintptr_t at = reinterpret_cast<uintptr_t>(proj) | reinterpret_cast<uintptr_t>(d->in_bias) | reinterpret_cast<uintptr_t>(d->q_norm_w) | reinterpret_cast<uintptr_t>(d->k_norm_w);
    if (!d->norm_full && ((d->D | d->V) & 7) == 0 && ((ld | d->q_col | d->k_col | d->v_col) & 3) == 0 && (at & 15) == 0 && (!d->rot_half || (np & 7) == 0)) {
        // as many blocks as eight an SM allow, or as a token has rows for
        const int most = (heads * lpr + 127) / 128, want = 148 * 8 / st->T, split = want < 1 ? 1 : (want < most ? want : most);
        const auto kernel = lpr == 4 ? kv4_prep_rows_kernel<4> : (lpr == 8 ? kv4_prep_rows_kernel<8> : kv4_prep_rows_kernel<16>);
        launch_chained(kernel, st->T * split, 128, (size_t)(2 * np) * sizeof(float), (cudaStream_t)stream, proj, ld, *st, *d, (uint8_t*)kpool, (uint8_t*)vpool, split, error_flag_dev());
        SEQ_LAUNCH_CHECK("attn_prep_kv4");
        return 0;
    }
    launch_chained(kv4_prep_kernel, st->T, 256, smem, (cudaStream_t)stream, proj, ld, *st, *d, (uint8_t*)kpool, (uint8_t*)vpool, Dmax, error_flag_dev());
    SEQ_LAUNCH_CHECK("attn_prep_kv4");
    return 0;
}

}  // extern "C"
