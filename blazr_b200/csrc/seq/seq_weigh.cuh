// seq_weigh.cuh -- what the kernels share that add up the soft-max weight of cached keys (seq_weigh.cu, seq_weigh_tc.cu)
#pragma once
#include "seq_attn.cuh"
#include "seq_kv4.cuh"

namespace b200seq {

struct WeighArgs {
    const float* q;            // query rows (pointer at the first head's column), stride ld
    int64_t ld;
    const float* kpool;        // f32 pages [page][row][G][D], or (four) 4-bit ones
    const uint8_t* kpool4;
    float* acc;                // [slots][G][acc_ld]
    int64_t acc_ld;
    int slots, H, G, D, NG;
    int last;                  // > 0: the last so many tokens of an entry count
    float scale, softcap;
    int chunk, window, keep_first;
    const float *head_scale, *sink;
    float* lse;                // f32 tiles: [T][H], base-2 logarithm of every row's sum of exponentials (minus infinity: nothing to give)
    float* part;               // work area of the path that is taken
    int key_blocks;            // rows' path: blocks of keys that the longest sequence may need, and as keys
    int64_t key_room;
    int64_t most_keys;         // of a sequence
    int* err;
};

constexpr float WEIGH_LOG2E = 1.4426950408889634f;

// the keys that a token at position p sees: lo .. p and those below keep
struct WeighSpan {
    int lo, p, keep;
    __device__ __forceinline__ WeighSpan(const WeighArgs& a, int pos) {
        p = pos, lo = a.chunk > 0 ? (pos / a.chunk) * a.chunk : 0, keep = a.window > 0 ? a.keep_first : 0;
        if (a.window > 0) lo = max(lo, pos - a.window + 1);
    }
    __device__ __forceinline__ bool sees(int j) const { return j <= p && (j >= lo || j < keep); }
};

// an entry as these kernels see it: its first token that counts (row of the step, place among the entry's), how many do, its keys; n = 0: none, or its keys have no place
struct WeighEntry {
    int t0, n, p0, keys, fresh, slot;      // p0: position of the first token that counts; keys: positions 0 .. keys - 1; fresh: the first position that this step brought
    __device__ __forceinline__ WeighEntry(const WeighArgs& a, const b200seq_step& st, int e, bool tell) {
        const int s0 = st.ent_start[e], s1 = st.ent_start[e + 1], len = s1 - s0;
        fresh = st.ent_pos0[e], slot = st.ent_slot[e];
        n = a.last > 0 && a.last < len ? a.last : len;
        t0 = s1 - n, keys = fresh + len, p0 = keys - n;
        const bool fine = s0 >= 0 && len >= 0 && s1 <= st.T && fresh >= 0 && slot >= 0 && slot < a.slots && keys <= a.acc_ld && keys <= a.most_keys && (keys + st.block_size - 1) / st.block_size <= st.max_blocks;
        if (!fine) {
            if (tell && len != 0) atomicOr(a.err, 1);
            n = 0;
        } else if (len == 0) {
            n = 0;
        }
    }
};

// score of a dot product in base 2: scaled, soft-capped
__device__ __forceinline__ float weigh_score(float dot, float factor, float softcap) {
    const float z = dot * factor;
    return softcap > 0.f ? softcap * WEIGH_LOG2E * tanhf(z / softcap) : z * WEIGH_LOG2E;
}
__device__ __forceinline__ float weigh_factor(const WeighArgs& a, int h) { return a.head_scale ? a.scale * a.head_scale[h] : a.scale; }

// base-2 logarithm of a row's denominator from its maximum and sum (base 2), with the sink's term
__device__ __forceinline__ float weigh_lse(const WeighArgs& a, int h, float m, float l) {
    if (a.sink) {
        const float sk = a.sink[h] * WEIGH_LOG2E, top = fmaxf(m, sk);
        l = (m == -INFINITY ? 0.f : l * exp2f(m - top)) + exp2f(sk - top), m = top;
    }
    return m == -INFINITY ? -INFINITY : m + log2f(l);
}

// one score by plain f32 products, for those that the split operands have no numbers for
__device__ __forceinline__ float weigh_key_at(const WeighArgs& a, int64_t row, const Kv4Row& r, int g, int d, bool four) {
    if (!four) return a.kpool[(row * a.G + g) * a.D + d];
    const uint32_t c = *reinterpret_cast<const uint32_t*>(a.kpool4 + r.codes + 4 * ((d % 32 / 8) * a.NG + d / 32)), par = *reinterpret_cast<const uint32_t*>(a.kpool4 + r.params + 4 * (d / 32));
    const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&par));
    return fmaf((float)((c >> (4 * (d % 8))) & 15u), sm.x, sm.y);
}
static __device__ __noinline__ float plain_score(const WeighArgs& a, const b200seq_step& st, const WeighEntry& en, int e, int g, int row, int key, bool four) {
    const int R = a.H / a.G, h = g * R + row % R, page = max(0, st.block_table[(int64_t)e * st.max_blocks + key / st.block_size]), o = key % st.block_size;
    const float* q = a.q + (int64_t)(en.t0 + row / R) * a.ld + (int64_t)h * a.D;
    const Kv4Row r = four ? kv4_row(page, o, st.block_size, g, a.G, a.NG) : Kv4Row{0, 0};
    float s = 0.f;
    for (int d = 0; d < a.D; ++d) s = fmaf(q[d], weigh_key_at(a, (int64_t)page * st.block_size + o, r, g, d, four), s);
    return weigh_score(s, weigh_factor(a, h), a.softcap);
}

// Steps of many rows on the tensor cores (seq_weigh_tc.cu): how a step is cut up and the work area it needs (from its host sizes alone), whether a layer's rows suit it, the launches
struct WeighTcPlan {
    int qtiles, stage;         // tiles of 64 split rows of a key head (bound), bytes of one
    int tiles, stat_parts;     // denominators: row tiles of 128 (bound), parts of a walk
    int key_tiles, parts;      // key tiles of 64 of the longest sequence; sums: parts of a walk
    int ne, ng;                // entries and key heads of a run
    int64_t key_room, q_floats, k_floats, lse_floats, stat_floats;
    size_t floats;
};
WeighTcPlan weigh_tc_plan(const b200seq_step& st, int H, int G, int D, int last, int64_t keys);
bool weigh_tc_takes(const WeighArgs& a, bool four);
int weigh_tc(const WeighArgs& a, const b200seq_step& st, const WeighTcPlan& p, float* scratch, bool four, cudaStream_t cs);

}  // namespace b200seq
