// seq_attn4.cuh -- arguments of the attend step over 4-bit pages, shared by its kernels
#pragma once
#include "seq_attn.cuh"
#include "seq_kv4.cuh"

namespace b200seq {

struct Attn4Args {
    const float* q;            // query rows (pointer at the first head's column), stride ld
    int64_t ld;
    int vec;                   // heads of whole 16-byte pieces
    const uint8_t *kpool, *vpool;
    int H, G, D, V, vdiv;      // key head g reads value head g / vdiv
    int Rb, HB, QT;            // query heads of a row tile, tiles a key head's query heads need, tokens of a row tile
    float scale;
    int chunk, window, keep_first;
    const float *head_scale, *sink, *gate;
    int64_t gld;
    int gated, gate_elem;
    float softcap;
    void* out;                 // [T, H * V]
    int out_dtype;
    int cluster;               // CTAs of a cluster that share a row tile's keys
    int tiles, heads;          // row tiles (bound), key heads * head blocks
    int parts;                 // tensor-core kernel: CTAs that share a row tile's keys
    float* part;               // work area.  Tensor-core kernel, parts > 1: [T][H][parts][V + 4] = maximum (base 2), sum, two unused, values
    int* err;
};

// the keys that rows at positions p0 .. hi can see, in tiles of KT positions: those of the kept first positions, then from the first visible one to hi
template <int KT>
struct KeySpan {
    int first, main0, total;
    __device__ __forceinline__ KeySpan(const Attn4Args& a, int p0, int hi) {
        int lo = a.chunk > 0 ? (p0 / a.chunk) * a.chunk : 0;
        if (a.window > 0) lo = max(lo, p0 - a.window + 1);
        const int keep = a.window > 0 ? a.keep_first : 0;
        first = (min(keep, lo) + KT - 1) / KT;
        main0 = max(lo / KT, first);
        total = first + hi / KT - main0 + 1;
    }
    __device__ __forceinline__ int key0(int tile) const { return (tile < first ? tile : main0 + tile - first) * KT; }
};

// one row's view: keys lo .. p and those below keep
struct RowSpan {
    int lo, p, keep;
    __device__ __forceinline__ RowSpan(const Attn4Args& a, int pos) {
        p = pos, lo = a.chunk > 0 ? (pos / a.chunk) * a.chunk : 0, keep = a.window > 0 ? a.keep_first : 0;
        if (a.window > 0) lo = max(lo, pos - a.window + 1);
    }
    __device__ __forceinline__ bool sees(int j) const { return j <= p && (j >= lo || j < keep); }
};

// Attend step of many rows on the tensor cores (seq_attn4_tc.cu)
struct Attn4TcPlan {
    int mt, Rb, HB, QT, parts;
    int64_t tiles, real;
};
bool attn4_tc_takes(int D, int V);
Attn4TcPlan attn4_tc_plan(const b200seq_step& st, int H, int G, int D, int V, int64_t keys);
cudaError_t attn4_tc_launch(Attn4Args a, const b200seq_step& st, const Attn4TcPlan& p, cudaStream_t cs);

}  // namespace b200seq
