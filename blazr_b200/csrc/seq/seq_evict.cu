// seq_evict.cu -- sequences cut back to the cached keys that were given the most weight: which ones (a choice for every layer and key head), and their rows moved together.
//
// Of an entry's n cached rows, n > keep, stay the first `first`, the last `recent` and the keep - first - recent of largest weight between them (ties: the lowest row); they go, in
// order, to the places 0 .. keep - 1.  The choice needs the weights alone: a block selects the smallest weight that stays by the bits of the ordered floats, eleven at a time, and
// writes the list of rows.  Moving is bound by the memory: every kept row is read and written once (keys, values, f32 or 4-bit codes with their parameters).
//
// A row never moves to a higher place.  So a block that walks over its rows (of one head, of a slice of their bytes) in chunks, all of a chunk read before any of it is written,
// may write into the pages that it reads: what it overwrites has been read, and nobody else touches these bytes.  That is what lets a cache be cut back where it lies.
#include "seq_kv4.cuh"

namespace b200seq {

namespace {

constexpr int LAYERS = 32;                // of one launch
constexpr int CHOOSE = 512;               // threads that choose
constexpr int EACH = 8;                   // neighbouring weights a thread lists at a time
constexpr int MOVE = 256;                 // threads that move

struct EvictArgs {
    uint8_t* pool[2][LAYERS];
    float* acc[LAYERS];
    int32_t* kept;                        // [layers][B][G][keep]
    const int32_t *slot, *rows, *bt, *to_slot, *to_bt;
    int64_t acc_ld;
    int layers, B, G, bs, mb, to_mb, slots, keep, first, recent;
    int units[2];                         // pieces of a row: keys, values
    int per[2];                           // pieces of a row that a block takes
    int slices;                           // blocks that share a head's rows
    int ng[2];                            // 4-bit pools: groups of a row
    int* err;
};

__device__ __forceinline__ uint32_t weight_key(float w) {      // whole numbers of the same order; NaN lowest
    if (w != w) return 0;
    const uint32_t b = __float_as_uint(w + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

// rows that entry e has and keeps; 0, 0: none, or it is not one
__device__ __forceinline__ void entry_rows(const EvictArgs& a, int e, int& n, int& kept, bool tell) {
    n = a.rows[e];
    const int s = a.slot[e], d = a.to_slot[e];
    const bool fine = n >= 0 && n <= a.acc_ld && (n + a.bs - 1) / a.bs <= a.mb && s >= 0 && s < a.slots && d >= 0 && d < a.slots && ((n < a.keep ? n : a.keep) + a.bs - 1) / a.bs <= a.to_mb;
    if (!fine) {
        if (tell) atomicOr(a.err, 1);
        n = 0;
    }
    kept = n < a.keep ? n : a.keep;
}

// grid (key heads, entries, layers)
__global__ void __launch_bounds__(CHOOSE) evict_choose_kernel(const __grid_constant__ EvictArgs a) {
    chain_enter();
    constexpr int WARPS = CHOOSE / 32;
    __shared__ unsigned hist[2048], wsum[WARPS], found[2];
    __shared__ uint2 tsum[WARPS];
    const int g = blockIdx.x, e = blockIdx.y, l = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int n, kept;
    entry_rows(a, e, n, kept, tid == 0 && g == 0 && l == 0);
    int32_t* list = a.kept + (((int64_t)l * a.B + e) * a.G + g) * a.keep;
    for (int i = kept + tid; i < a.keep; i += CHOOSE) list[i] = -1;
    if (n == 0) return;
    const float* w = a.acc[l] + ((int64_t)a.slot[e] * a.G + g) * a.acc_ld;
    float* to = a.acc[l] + ((int64_t)a.to_slot[e] * a.G + g) * a.acc_ld;
    if (n <= a.keep) {
        for (int i = tid; i < n; i += CHOOSE) {
            list[i] = i;
            if (to != w) to[i] = w[i];
        }
        return;
    }
    const int lo = a.first, hi = n - a.recent;              // the rows between: more than are chosen of them
    unsigned least = 0xffffffffu, ties = 0;                 // keys above stay, and the first `ties` equal ones
    if (a.keep > a.first + a.recent) {
        unsigned want = (unsigned)(a.keep - a.first - a.recent), prefix = 0;
        for (int level = 0; level < 3; ++level) {
            const int bits = level < 2 ? 11 : 10, shift = level == 0 ? 21 : level == 1 ? 10 : 0;
            for (int i = tid; i < 2048; i += CHOOSE) hist[i] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += CHOOSE) {
                const unsigned k = weight_key(w[i]);
                if (level == 0 || (k >> (shift + bits)) == prefix) atomicAdd(hist + ((k >> shift) & ((1u << bits) - 1)), 1u);
            }
            __syncthreads();
            // bins 4 t .. 4 t + 3 of thread t, added up from the top
            unsigned b[4], s = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = hist[4 * tid + j], s += b[j];
            unsigned up = s;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_down_sync(0xffffffffu, up, o);
                if (lane + o < 32) up += y;
            }
            if (lane == 0) wsum[warp] = up;
            __syncthreads();
            for (int k = warp + 1; k < WARPS; ++k) up += wsum[k];
            unsigned over = up - s;
#pragma unroll
            for (int j = 3; j >= 0; --j) {
                if (over < want && over + b[j] >= want) found[0] = 4 * tid + j, found[1] = over;
                over += b[j];
            }
            __syncthreads();
            prefix = level == 0 ? found[0] : (prefix << bits) | found[0];
            want -= found[1];
            __syncthreads();
        }
        least = prefix, ties = want;
    }
    // the list, in order: a tile of rows at a time, all of it read before its places are written
    unsigned at = 0, equal = 0;
    for (int t0 = 0; t0 < n; t0 += CHOOSE * EACH) {
        float x[EACH];
        bool stay[EACH], eq[EACH];
        unsigned above = 0, same = 0;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int i = t0 + tid * EACH + j;
            x[j] = i < n ? w[i] : 0.f;
            const unsigned k = weight_key(x[j]);
            const bool mid = i >= lo && i < hi;
            stay[j] = i < n && (!mid || k > least), eq[j] = mid && k == least;
            above += stay[j], same += eq[j];
        }
        uint2 s = make_uint2(above, same);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, s.x, o), z = __shfl_up_sync(0xffffffffu, s.y, o);
            if (lane >= o) s.x += y, s.y += z;
        }
        if (lane == 31) tsum[warp] = s;
        __syncthreads();
        uint2 before = make_uint2(0, 0), all = make_uint2(0, 0);
        for (int k = 0; k < WARPS; ++k) {
            const uint2 y = tsum[k];
            if (k < warp) before.x += y.x, before.y += y.y;
            all.x += y.x, all.y += y.y;
        }
        // rows of equal weight stay while there is room for them: `ties` of the entry's
        unsigned eqs = equal + before.y + s.y - same, place = at + before.x + s.x - above + min(eqs, ties);
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const bool in = stay[j] || (eq[j] && eqs < ties);
            if (in) {
                list[place] = t0 + tid * EACH + j;
                to[place] = x[j];
                ++place;
            }
            eqs += eq[j];
        }
        at += all.x, equal += all.y;
        // (`at` counts the rows above; equal ones that stay are in `place` through eqs)
        __syncthreads();
    }
}

template <class V>
__device__ __forceinline__ V load_piece(const uint8_t* p) { return *reinterpret_cast<const V*>(p); }

// where piece u of row o of page p of head g begins.  f32: pieces of sizeof(V) of rows [page][row][head]; 4 bits: five pieces of 4 NG bytes, four of codes, one of parameters
template <class V, bool FOUR>
__device__ __forceinline__ int64_t piece_at(const EvictArgs& a, int kv, int page, int o, int g, int u) {
    if (FOUR) {
        const Kv4Row r = kv4_row(page, o, a.bs, g, a.G, a.ng[kv]);
        return u < 4 ? r.codes + u * 4 * a.ng[kv] : r.params;
    }
    return ((((int64_t)page * a.bs + o) * a.G + g) * a.units[kv] + u) * (int64_t)sizeof(V);
}

// grid (slices of a row, entries * key heads, layers): one block moves its pieces of all rows, in chunks
template <class V, bool FOUR>
__global__ void __launch_bounds__(MOVE) evict_move_kernel(const __grid_constant__ EvictArgs a, int kv) {
    chain_enter();
    constexpr int ITEMS = 4, SPAN = MOVE * ITEMS, ROWS = SPAN / 2;
    // (page, row of the page) of a chunk's rows; page < 0: the row stays where it is.  Three of each: the next chunk's are looked up while slower warps still write the last one.
    __shared__ int2 from[3][ROWS], dest[3][ROWS];
    const int u0 = blockIdx.x * a.per[kv], per = min(a.per[kv], a.units[kv] - u0), e = blockIdx.y / a.G, g = blockIdx.y - e * a.G, l = blockIdx.z, tid = threadIdx.x;
    if (per <= 0) return;
    int n, kept;
    entry_rows(a, e, n, kept, false);
    const int32_t* list = a.kept + (((int64_t)l * a.B + e) * a.G + g) * a.keep;
    const int32_t *bt = a.bt + (int64_t)e * a.mb, *to = a.to_bt + (int64_t)e * a.to_mb;
    uint8_t* pool = a.pool[kv][l];
    const int rows = min(SPAN / per, ROWS);                 // of a chunk
    auto look = [&](int r0, int b) {
        for (int i = tid; i < rows && r0 + i < kept; i += MOVE) {
            const int src = list[r0 + i], dst = r0 + i;
            int sp = -1, dp = -1;
            if (src >= 0 && src < n) {
                sp = bt[src / a.bs], dp = to[dst / a.bs];
                if (sp < 0 || dp < 0) {
                    if (l == 0 && kv == 0 && blockIdx.x == 0) atomicOr(a.err, 1);
                    sp = -1;
                }
            }
            if (sp == dp && src == dst) sp = -1;
            from[b][i] = make_int2(sp, src % a.bs), dest[b][i] = make_int2(dp, dst % a.bs);
        }
    };
    look(0, 0);
    __syncthreads();
    int b = 0;
    for (int r0 = 0; r0 < kept; r0 += rows, b = b == 2 ? 0 : b + 1) {
        const int m = min(rows, kept - r0) * per;
        V x[ITEMS];
        bool go[ITEMS];
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int i = k * MOVE + tid;
            go[k] = false;
            if (i < m) {
                const int r = i / per, u = u0 + i - r * per;
                const int2 s = from[b][r];
                go[k] = s.x >= 0;
                if (go[k]) x[k] = load_piece<V>(pool + piece_at<V, FOUR>(a, kv, s.x, s.y, g, u));
            }
        }
        if (r0 + rows < kept) look(r0 + rows, b == 2 ? 0 : b + 1);
        __syncthreads();                                    // all of the chunk has been read
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            if (!go[k]) continue;
            const int i = k * MOVE + tid, r = i / per, u = u0 + i - r * per;
            const int2 d = dest[b][r];
            *reinterpret_cast<V*>(pool + piece_at<V, FOUR>(a, kv, d.x, d.y, g, u)) = x[k];
        }
    }
}

template <class V, bool FOUR>
cudaError_t move(EvictArgs& a, int kv, int piece, cudaStream_t cs) {
    // Blocks walk over their rows one chunk after another, so that the more of them share a row's bytes the sooner they are through: down to 32 bytes of a row each.
    const int64_t heads = (int64_t)a.B * a.G * a.layers;
    const int least = piece >= 32 ? 1 : 32 / piece, most = FOUR ? 1 : (a.units[kv] + least - 1) / least;
    int64_t slices = (4 * 148 + heads - 1) / heads;
    slices = slices < most ? slices : most;
    a.per[kv] = FOUR ? a.units[kv] : (int)((a.units[kv] + slices - 1) / slices);
    if (a.per[kv] > MOVE) a.per[kv] = MOVE;
    const int blocks = (a.units[kv] + a.per[kv] - 1) / a.per[kv];
    launch_chained(evict_move_kernel<V, FOUR>, dim3(blocks, a.B * a.G, a.layers), MOVE, 0, cs, a, kv);
    return cudaGetLastError();
}

}  // namespace

}  // namespace b200seq

using namespace b200seq;

extern "C" int b200seq_evict_keys(void* const* kpools, void* const* vpools, float* const* accs, int layers, int kv_bits, int block_size, int G, int D, int Gv, int V,
                                  int slots, int64_t acc_ld, const int32_t* slot, const int32_t* rows, const int32_t* table, int max_blocks, const int32_t* to_slot,
                                  const int32_t* to_table, int to_max_blocks, int B, int keep, int first, int recent, int32_t* kept, void* stream) {
    if (layers < 0 || B < 0 || block_size < 1 || G < 1 || D < 1 || Gv < 1 || V < 1 || slots < 1 || acc_ld < 1 || max_blocks < 1 || to_max_blocks < 1 || (kv_bits != 4 && kv_bits != 32))
        return fail(B200SEQ_ERR_INVALID_ARG, "evict_keys: bad sizes");
    if (keep < 1 || first < 0 || recent < 0 || (int64_t)first + recent > keep) return fail(B200SEQ_ERR_INVALID_ARG, "evict_keys: the first %d and the last %d rows are more than the %d to keep", first, recent, keep);
    if (Gv != G) return fail(B200SEQ_ERR_UNSUPPORTED, "evict_keys: %d key heads choose for themselves, their rows of %d value heads do not go apart", G, Gv);
    if (layers > 0 && B > 0 && (!kpools || !vpools || !accs || !slot || !rows || !table || !to_slot || !to_table || !kept)) return fail(B200SEQ_ERR_INVALID_ARG, "evict_keys: null arrays");
    if (kv_bits == 4 && (D > KV4_MAX_DIM || V > KV4_MAX_DIM || !kv4_pages_fit(block_size, G, D > V ? D : V)))
        return fail(B200SEQ_ERR_UNSUPPORTED, "evict_keys: 4-bit pages hold heads of up to %d values", KV4_MAX_DIM);
    if ((int64_t)B * G > 65535 || B > 65535 || D > (1 << 20) || V > (1 << 20)) return fail(B200SEQ_ERR_UNSUPPORTED, "evict_keys: up to 65535 heads of all entries");
    for (int i = 0; i < layers; ++i)
        if (!kpools[i] || !vpools[i] || !accs[i] || (kv_bits == 4 && ((reinterpret_cast<uintptr_t>(kpools[i]) | reinterpret_cast<uintptr_t>(vpools[i])) & 15)))
            return fail(B200SEQ_ERR_INVALID_ARG, "evict_keys: a pool of layer %d is null or not on a 16-byte boundary", i);
    const cudaStream_t cs = (cudaStream_t)stream;
    for (int l0 = 0; l0 < layers && B > 0; l0 += LAYERS) {
        EvictArgs a = {};
        a.layers = layers - l0 < LAYERS ? layers - l0 : LAYERS;
        bool wide[2] = {(D & 3) == 0, (V & 3) == 0};
        for (int i = 0; i < a.layers; ++i) {
            a.pool[0][i] = (uint8_t*)kpools[l0 + i], a.pool[1][i] = (uint8_t*)vpools[l0 + i], a.acc[i] = accs[l0 + i];
            for (int kv = 0; kv < 2; ++kv) wide[kv] = wide[kv] && (reinterpret_cast<uintptr_t>(a.pool[kv][i]) & 15) == 0;
        }
        a.kept = kept + (int64_t)l0 * B * G * keep;
        a.slot = slot, a.rows = rows, a.bt = table, a.to_slot = to_slot, a.to_bt = to_table, a.acc_ld = acc_ld;
        a.B = B, a.G = G, a.bs = block_size, a.mb = max_blocks, a.to_mb = to_max_blocks, a.slots = slots, a.keep = keep, a.first = first, a.recent = recent, a.err = error_flag_dev();
        launch_chained(evict_choose_kernel, dim3(G, B, a.layers), CHOOSE, 0, cs, a);
        SEQ_LAUNCH_CHECK("evict_keys");
        for (int kv = 0; kv < 2; ++kv) {
            const int size = kv ? V : D;
            cudaError_t err;
            if (kv_bits == 4) {
                a.ng[kv] = kv4_groups(size), a.units[kv] = 5;
                err = a.ng[kv] == 4 ? move<uint4, true>(a, kv, 16, cs) : a.ng[kv] == 2 ? move<uint2, true>(a, kv, 8, cs) : move<uint32_t, true>(a, kv, 4, cs);
            } else {
                a.units[kv] = wide[kv] ? size / 4 : size;
                err = wide[kv] ? move<uint4, false>(a, kv, 16, cs) : move<uint32_t, false>(a, kv, 4, cs);
            }
            if (err != cudaSuccess) return cuda_status(err, "evict_keys");
            count_launch();
        }
    }
    return 0;
}
