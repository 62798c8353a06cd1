// seq_kv4.cuh -- KV pages held in 4 bits: the layout of a page, and how 32 values become codes.
//
// A row of D values (one position, one head) is NG = 1, 2 or 4 groups of 32 (D <= 32, 64, 128; places behind D are held as zero).  A group has a minimum m and a
// step s, both f16, and a 4-bit code per value, which stands for m + s * code:
//   m = f16(min x),  s = (max x - m) * (1 / 15) rounded up to 7 significant bits and to a multiple of 2^-24,  code = clamp(rint((x - m) * (1 / s)), 0, 15)
// (1 / 15 is the f32 number below it, so that a range of fifteen whole steps keeps its step).  Seven bits, because s * code is then an f16 number (7 + 4 bits): the
// tensor cores multiply what the cache holds with no further rounding.  It costs a step that is up to 1.6 % wider; a minimum beside it
// serves keys, whose channels do not lie around zero.  Values are limited to +-32000 (15 s stays an f16 number), NaN is held as 0; either raises bit 3 of the error flags.
//
// Bytes of a pool: [page][head][segment], so that one head's rows of a page are consecutive (10 NG 16-byte pieces a unit of 16 rows: one request of a warp or
// two).  A segment is cut into units of 16 rows (block sizes that are not a multiple of 16: one unit of all rows), each unit holds its rows' codes (16 NG
// bytes a row), then its rows' (s, m) pairs (4 NG bytes a row).  Order of a row's codes, low 4 bits first:
//   keys    32-bit words [part c < 4][group],  eight values 32 group + 8 c + i:  thread c of a quad reads its words of all groups in one piece
//   values  16-bit words [part r < 8][group],  four values 32 group + 4 r + i:   the eight threads that hold a column of the product each, likewise
#pragma once
#include <cuda_fp16.h>

#include "seq_common.cuh"

namespace b200seq {

constexpr int KV4_MAX_DIM = 128;
constexpr int KV4_ERR_RANGE = 8;         // error flag: a value that is not a number within +-32000 was stored
constexpr float KV4_LIMIT = 32000.f;
constexpr float KV4_FIFTEENTH = 0x1.11111p-4f;

__host__ __device__ __forceinline__ int kv4_groups(int D) { return D <= 32 ? 1 : (D <= 64 ? 2 : 4); }
__host__ __device__ __forceinline__ int kv4_unit(int bs) { return bs % 16 == 0 ? 16 : bs; }

// row `o` of a page of `bs` rows, head g of G: offset of its codes and of its parameters in the pool (pages of less than 2 GiB: checked by the callers)
struct Kv4Row {
    int64_t codes, params;
};
__device__ __forceinline__ Kv4Row kv4_row(int page, int o, int bs, int g, int G, int NG) {
    const int unit = kv4_unit(bs), u = unit == 16 ? o >> 4 : 0, ru = unit == 16 ? o & 15 : o, head = bs * NG * 20;   // (o < bs)
    const int64_t base = (int64_t)page * (G * head) + (g * head + u * (unit * NG * 20));
    return Kv4Row{base + ru * NG * 16, base + (unit * NG * 16 + ru * NG * 4)};
}
inline bool kv4_pages_fit(int bs, int heads, int D) { return (int64_t)bs * heads * kv4_groups(D) * 20 <= 0x7fffffff; }

// an entry of a block table; a negative one is no page: the first page's memory is read in its place, and the error flag says so
__device__ __forceinline__ int kv4_page_read(int page, int* err) {
    if (page < 0) atomicOr(err, 1);
    return max(page, 0);
}

// A group of 32 values, eight in each of four neighbouring lanes (`n` of the lane's eight are values of the row, the rest do not exist).  Returns the lane's eight
// codes, the first in the lowest bits, and, the same in all four lanes, the (s, m) pair.  Every lane of the warp takes part.
__device__ __forceinline__ uint32_t kv4_quantise(float (&x)[8], int n, uint32_t& param, bool& odd) {
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) fine &= fabsf(x[i]) <= KV4_LIMIT;      // (places that do not exist hold zeros)
    if (!fine) {
        odd = true;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -KV4_LIMIT), KV4_LIMIT);
    }
    if (n < 8) {
#pragma unroll
        for (int i = 1; i < 8; ++i) x[i] = i < n ? x[i] : x[0];
    }
    float lo = fminf(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), fminf(fminf(x[4], x[5]), fminf(x[6], x[7])));
    float hi = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    if (n == 0) lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o)), hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    if (!(lo <= hi)) {   // a group behind the row's end
        param = 0;
        return 0;
    }
    const __half mh = __float2half_rn(lo);
    const float m = __half2float(mh);
    float s = fmaxf((hi - m) * KV4_FIFTEENTH, 0.f);
    s = __uint_as_float((__float_as_uint(s) + 0x1FFFFu) & ~0x1FFFFu);
    if (s < 0x1p-18f) s = ceilf(s * 0x1p24f) * 0x1p-24f;
    param = (uint32_t)__half_as_ushort(__float2half_rn(s)) | ((uint32_t)__half_as_ushort(mh) << 16);
    const float inv = s > 0.f ? 1.0f / s : 0.f;
    // rint(y) for y in 0 .. 15 by adding 1.5 2^23, whose bits then end in the number; the words of eight of them add up, sixteenfold each, to the codes and a constant
    uint32_t w = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) w = w * 16u + __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(x[i] - m, inv), 0.f), 15.f), 12582912.f));
    w -= 0x4B400000u * 0x11111111u;
    return n < 8 ? w & ((1u << (4 * n)) - 1u) : w;
}

// The place of a lane's codes in a row's: lane hl holds values 8 hl .. 8 hl + 7, of group hl / 4: one word of a key row, two 16-bit words of a value row
__device__ __forceinline__ int kv4_key_place(int hl, int NG) { return ((hl & 3) * NG + (hl >> 2)) * 4; }
__device__ __forceinline__ int kv4_value_place(int hl, int NG) { return (2 * (hl & 3) * NG + (hl >> 2)) * 2; }   // (the second: 2 NG bytes on)

}  // namespace b200seq
