// seq_evict.cu -- sequences cut back to the cached keys that were given the most weight: which ones (a choice for every layer and key head), and their rows moved together.
//
// Of an entry's n cached rows, n > keep, stay the first `first`, the last `recent` and the keep - first - recent of largest weight between them (ties: the lowest row); they go, in
// order, to the places 0 .. keep - 1.  The choice needs the weights alone: a block selects the smallest weight that stays by the bits of the ordered floats, eleven at a time, and
// writes the list of rows.  Moving is bound by the memory: every kept row is read and written once (keys, values, f32 or 4-bit codes with their parameters).
//
// A row never moves to a higher place.  So whoever walks over a head's rows in chunks, all of a chunk read before any of it is written, may write into the pages that it reads: what
// it overwrites has been read, and nobody else touches these bytes.  That is what lets a cache be cut back where it lies.  A cluster of up to eight CTAs walks together, each with
// whole rows of a chunk, and waits for all of them between reading and writing; the next chunks are on their way by then.  The wait orders those reads before those writes: a barrier of the
// block where it is alone, else a barrier of the cluster with release and acquire.  A release waits for all that its thread has under way, so that one warp that moves nothing does it
// for its block (two sequences of 32768 rows in place, in all: 415 us; with a release of every thread that reads 436 to 590, with none, so in no order that memory promises, 397).  Two
// sequences of 32768 rows to 16384, 8 heads of 128, four layers: 390 us of moving, 5.5 TB/s.  (Pages and kept rows in any order take the same time: what it cost before were instructions for addresses.)
#include "seq_kv4.cuh"

namespace b200seq {

namespace {

constexpr int LAYERS = 32;                // of one launch
constexpr int EACH = 8;                   // weights a thread lists at a time
constexpr int HELD = 49152;               // weights that a block has in shared memory; longer rows are read four times
constexpr int MOVE = 256;                 // threads that move (and a warp that arrives for them, in clusters)
// Pieces of a chunk a thread has, chunks on their way, rows looked up at a time.  Small ones, so that many CTAs share an SM; in clusters larger ones, as each costs a barrier.  Eight
// sequences of 2301 rows in 16 layers of 4-bit pages (blocks alone) 160 us, with four pieces 172; two of 32768 in four layers of f32 pages (clusters of four) 415, with two pieces 447
constexpr int ITEMS_ALONE = 2, ITEMS_CLUSTER = 4, STAGES = 2, BATCH = 512;

struct EvictArgs {
    uint8_t* pool[2][LAYERS];
    float* acc[LAYERS];
    int32_t* kept;                        // [layers][B][G][keep]
    const int32_t *slot, *rows, *bt, *to_slot, *to_bt;
    int64_t acc_ld;
    int layers, B, G, bs, mb, to_mb, slots, keep, first, recent;
    int units[2];                         // pieces of a row: keys, values
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

// grid (key heads, entries, layers).  Dynamic shared memory: as many weights as a slot has room for, or HELD
template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_choose_kernel(const __grid_constant__ EvictArgs a) {
    chain_enter();
    constexpr int WARPS = THREADS / 32, PER = 2048 / THREADS;
    extern __shared__ __align__(16) float held[];
    __shared__ unsigned hist[2048], wsum[WARPS], found[2];
    __shared__ uint2 tsum[2][WARPS];
    const int g = blockIdx.x, e = blockIdx.y, l = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int n, kept;
    entry_rows(a, e, n, kept, tid == 0 && g == 0 && l == 0);
    int32_t* list = a.kept + (((int64_t)l * a.B + e) * a.G + g) * a.keep;
    for (int i = kept + tid; i < a.keep; i += THREADS) list[i] = -1;
    if (n == 0) return;
    const float* w = a.acc[l] + ((int64_t)a.slot[e] * a.G + g) * a.acc_ld;
    float* to = a.acc[l] + ((int64_t)a.to_slot[e] * a.G + g) * a.acc_ld;
    if (n <= a.keep) {
        for (int i = tid; i < n; i += THREADS) {
            list[i] = i;
            if (to != w) to[i] = w[i];
        }
        return;
    }
    const bool here = n <= HELD;
    if (here) {
#pragma unroll 8
        for (int i = tid; i < n; i += THREADS) held[i] = w[i];
    }
    const float* src = here ? held : w;
    const int lo = a.first, hi = n - a.recent;              // the rows between: more than are chosen of them
    unsigned least = 0xffffffffu, ties = 0;                 // keys above stay, and the first `ties` equal ones
    if (a.keep > a.first + a.recent) {
        unsigned want = (unsigned)(a.keep - a.first - a.recent), prefix = 0;
        for (int level = 0; level < 3; ++level) {
            const int bits = level < 2 ? 11 : 10, shift = level == 0 ? 21 : level == 1 ? 10 : 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) hist[tid + i * THREADS] = 0;
            __syncthreads();
#pragma unroll 8
            for (int i = lo + tid; i < hi; i += THREADS) {
                const unsigned k = weight_key(src[i]);
                if (level == 0 || (k >> (shift + bits)) == prefix) atomicAdd(hist + ((k >> shift) & ((1u << bits) - 1)), 1u);
            }
            __syncthreads();
            // bins PER t .. of thread t, added up from the top
            unsigned b[PER], s = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) b[j] = hist[PER * tid + j], s += b[j];
            unsigned up = s;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_down_sync(0xffffffffu, up, o);
                if (lane + o < 32) up += y;
            }
            if (lane == 0) wsum[warp] = up;
            __syncthreads();
            unsigned over = up - s;
            for (int k = warp + 1; k < WARPS; ++k) over += wsum[k];
#pragma unroll
            for (int j = PER - 1; j >= 0; --j) {
                if (over < want && over + b[j] >= want) found[0] = PER * tid + j, found[1] = over;
                over += b[j];
            }
            __syncthreads();
            prefix = level == 0 ? found[0] : (prefix << bits) | found[0];
            want -= found[1];
        }
        least = prefix, ties = want;
    }
    __syncthreads();                                        // (the weights have been read, and held ones are in place)
    // the list, in order: a tile of rows at a time, all of it read before its places are written
    unsigned at = 0, equal = 0;                             // of the tiles before: rows that stay whatever their rank, rows of weight `least`
    int buf = 0;
    for (int t0 = 0; t0 < n; t0 += THREADS * EACH, buf ^= 1) {
        // a warp has EACH * 32 neighbouring rows, 32 of them at a time: what stays of those goes to neighbouring places
        float x[EACH];
        unsigned stay[EACH], eq[EACH], above = 0, same = 0;
        const int i0 = t0 + warp * (EACH * 32) + lane;
#pragma unroll
        for (int j = 0; j < EACH; ++j) x[j] = i0 + 32 * j < n ? src[i0 + 32 * j] : 0.f;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int i = i0 + 32 * j;
            const unsigned k = weight_key(x[j]);
            const bool mid = i >= lo && i < hi;
            stay[j] = __ballot_sync(0xffffffffu, i < n && (!mid || k > least)), eq[j] = __ballot_sync(0xffffffffu, mid && k == least);
            above += __popc(stay[j]), same += __popc(eq[j]);
        }
        if (lane == 0) tsum[buf][warp] = make_uint2(above, same);
        __syncthreads();
        uint2 before = make_uint2(0, 0), all = make_uint2(0, 0);
        for (int k = 0; k < WARPS; ++k) {
            const uint2 y = tsum[buf][k];
            if (k < warp) before.x += y.x, before.y += y.y;
            all.x += y.x, all.y += y.y;
        }
        // rows of equal weight stay while there is room for them: `ties` of the entry's
        unsigned over = at + before.x, eqs = equal + before.y;
        const unsigned below = (1u << lane) - 1u;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const unsigned my = eqs + __popc(eq[j] & below);
            if (((stay[j] >> lane) & 1u) || (((eq[j] >> lane) & 1u) && my < ties)) {
                const unsigned place = over + __popc(stay[j] & below) + min(my, ties);
                list[place] = i0 + 32 * j;
                to[place] = x[j];
            }
            over += __popc(stay[j]), eqs += __popc(eq[j]);
        }
        at += all.x, equal += all.y;
    }
}

// Where a row begins in a pool.  f32: pieces of sizeof(V) of rows [page][row][head]; 4 bits: five pieces of 4 NG bytes, four of codes, and one of parameters `params` further on
struct RowAt {
    int64_t at;
    int params;
};
template <class V, bool FOUR>
__device__ __forceinline__ RowAt row_at(const EvictArgs& a, int kv, int page, int o, int g) {
    if (FOUR) {
        const Kv4Row r = kv4_row(page, o, a.bs, g, a.G, a.ng[kv]);
        return RowAt{r.codes, (int)(r.params - r.codes)};
    }
    return RowAt{(((int64_t)page * a.bs + o) * a.G + g) * (a.units[kv] * (int64_t)sizeof(V)), 0};
}

template <class V>
__device__ __forceinline__ void copy_in(V* dst, const uint8_t* src) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    if (sizeof(V) == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(sizeof(V)) : "memory");
}

// grid (cluster, entries * key heads, layers [* keys and values]).  BOTH: keys and values are of one size.  ALONE: the cluster is one block
template <class V, bool FOUR, bool BOTH, bool ALONE>
__global__ void __launch_bounds__(ALONE ? MOVE : MOVE + 32) evict_move_kernel(const __grid_constant__ EvictArgs a, int which) {
    chain_enter();
    constexpr int ITEMS = ALONE ? ITEMS_ALONE : ITEMS_CLUSTER, SPAN = MOVE * ITEMS;
    extern __shared__ __align__(16) uint8_t ring_raw[];
    V* const ring = reinterpret_cast<V*>(ring_raw);
    // Where the rows of two batches lie and go (from < 0: the row stays where it is).  Looked up a batch ahead, four chunks or more: the chain list, page takes as long as two of
    // them; and as addresses, since made again for every piece they were what the kernel spent its time on (2.3 us a chunk of 16 KB, whatever the rows' order)
    __shared__ int64_t from[2 * BATCH], dest[2 * BATCH];
    __shared__ int from_par[FOUR ? 2 * BATCH : 1], dest_par[FOUR ? 2 * BATCH : 1];
    const int kv = BOTH ? (int)blockIdx.z & 1 : which, l = BOTH ? (int)blockIdx.z >> 1 : blockIdx.z;
    const int per = a.units[kv], e = blockIdx.y / a.G, g = blockIdx.y - e * a.G, tid = threadIdx.x, rank = blockIdx.x, ranks = gridDim.x;
    int n, kept;
    entry_rows(a, e, n, kept, false);
    const int32_t* list = a.kept + (((int64_t)l * a.B + e) * a.G + g) * a.keep;
    const int32_t *bt = a.bt + (int64_t)e * a.mb, *to = a.to_bt + (int64_t)e * a.to_mb;
    uint8_t* pool = a.pool[kv][l];
    // a chunk is `rows` rows of every CTA of the cluster, a batch K chunks; rows of more than SPAN pieces go in several runs over them
    const int span = min(per, SPAN), rows = min(SPAN / span, BATCH / STAGES), K = BATCH / rows, step = rows * ranks;
    auto look = [&](int batch, int at) {
        for (int i = tid; i < K * rows; i += MOVE) {
            const int c = i / rows, dst = (batch * K + c) * step + rank * rows + i - c * rows;
            if (dst >= kept) continue;
            const int src = list[dst];
            int sp = -1, dp = -1;
            if (src >= 0 && src < n) {
                sp = bt[src / a.bs], dp = to[dst / a.bs];
                if (sp < 0 || dp < 0) {
                    if (l == 0 && kv == 0) atomicOr(a.err, 1);
                    sp = -1;
                }
            }
            const RowAt f = row_at<V, FOUR>(a, kv, max(sp, 0), src < 0 ? 0 : src % a.bs, g), t = row_at<V, FOUR>(a, kv, max(dp, 0), dst % a.bs, g);
            from[at + i] = sp < 0 || f.at == t.at ? -1 : f.at, dest[at + i] = t.at;
            if (FOUR) from_par[at + i] = f.params, dest_par[at + i] = t.params;
        }
    };
    const int chunks = (kept + step - 1) / step;
    if (!ALONE && tid >= MOVE) {      // (a warp of its own)
        for (int u0 = 0; u0 < per; u0 += span)
            for (int c = 0; c < chunks; ++c) {
                asm volatile("bar.sync 2, %0;" ::"n"(MOVE + 32) : "memory");
                asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            }
        return;
    }
    auto movers = []() { asm volatile("bar.sync 1, %0;" ::"n"(MOVE) : "memory"); };
    for (int u0 = 0; u0 < per; u0 += span) {
        int pr[ITEMS], pu[ITEMS];                           // a thread's pieces of a chunk: row, byte (FOUR: piece) of the row
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int i = k * MOVE + tid;
            pr[k] = i / span;
            const int u = u0 + i - pr[k] * span;
            if (pr[k] >= rows || u >= per) pr[k] = 0x3fffffff;
            pu[k] = FOUR && u == 4 ? -1 : u * (int)sizeof(V);
        }
        // a thread's pieces of a chunk go through its own places of the ring
        auto load = [&](int at, int left, int stage) {      // at: the chunk's first place in the tables; left: rows from this CTA's first one on
            V* const to_ring = ring + stage * SPAN + tid;
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (pr[k] >= left) continue;
                const int64_t f = from[at + pr[k]];
                if (f >= 0) copy_in(to_ring + k * MOVE, pool + f + (FOUR && pu[k] < 0 ? from_par[at + pr[k]] : pu[k]));
            }
        };
        auto store = [&](int at, int left, int stage) {
            const V* const of_ring = ring + stage * SPAN + tid;
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (pr[k] >= left || from[at + pr[k]] < 0) continue;
                *reinterpret_cast<V*>(pool + dest[at + pr[k]] + (FOUR && pu[k] < 0 ? dest_par[at + pr[k]] : pu[k])) = of_ring[k * MOVE];
            }
        };
        const int mine = kept - rank * rows;
        int load_at = 0, store_at = 0, load_stage = 0, store_stage = 0, in_batch = 0, batch = 0;
        auto load_next = [&](int c) {
            if (c < chunks) load(load_at, mine - c * step, load_stage);
            asm volatile("cp.async.commit_group;" ::: "memory");
            load_at += rows, load_stage = load_stage + 1 == STAGES ? 0 : load_stage + 1;
            if (load_at >= 2 * K * rows) load_at = 0;
        };
        movers();
        look(0, 0);
        movers();
        for (int c = 0; c < STAGES - 1; ++c) load_next(c);
        for (int c = 0; c < chunks; ++c) {
            load_next(c + STAGES - 1);                      // rows from the end of this chunk on: nothing that this one or an earlier one writes
            // all of this chunk has been read, by all CTAs, before any of it is written
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            if (ALONE) {
                movers();
            } else {
                asm volatile("bar.arrive 2, %0;" ::"n"(MOVE + 32) : "memory");
                asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            }
            store(store_at, mine - c * step, store_stage);
            store_at += rows, store_stage = store_stage + 1 == STAGES ? 0 : store_stage + 1;
            if (store_at >= 2 * K * rows) store_at = 0;
            if (in_batch == 0) {                            // (whoever wrote by the batch before this one is through)
                look(batch + 1, (batch + 1) & 1 ? K * rows : 0);
                movers();
            }
            if (++in_batch == K) in_batch = 0, ++batch;
        }
    }
}

template <class V, bool FOUR, bool BOTH, bool ALONE>
cudaError_t move_as(const EvictArgs& a, int kv, int cluster, cudaStream_t cs) {
    const int smem = STAGES * MOVE * (ALONE ? ITEMS_ALONE : ITEMS_CLUSTER) * (int)sizeof(V);
    const cudaError_t e = cudaFuncSetAttribute(evict_move_kernel<V, FOUR, BOTH, ALONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension, attr[1].val.clusterDim.x = cluster, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(cluster, a.B * a.G, a.layers * (BOTH ? 2 : 1)), cfg.blockDim = ALONE ? MOVE : MOVE + 32, cfg.dynamicSmemBytes = smem, cfg.stream = cs, cfg.attrs = attr;
    cfg.numAttrs = ALONE ? 1 : 2;
    cudaLaunchKernelEx(&cfg, evict_move_kernel<V, FOUR, BOTH, ALONE>, a, kv);
    return cudaGetLastError();
}
template <class V, bool FOUR, bool BOTH>
cudaError_t move_as(const EvictArgs& a, int kv, cudaStream_t cs) {
    const int64_t heads = (int64_t)a.B * a.G * a.layers * (BOTH ? 2 : 1);
    // Three CTAs an SM, where a head's rows are enough for so many (128 heads: clusters of 1, 2, 4 took 785, 542, 411 us; 2048 heads: 143, 143, 157; before the blocks' order was asked for)
    int cluster = 1;
    while (cluster < 8 && heads * cluster < 3 * 148) cluster *= 2;
    return cluster == 1 ? move_as<V, FOUR, BOTH, true>(a, kv, 1, cs) : move_as<V, FOUR, BOTH, false>(a, kv, cluster, cs);
}
template <class V, bool FOUR>
cudaError_t move(const EvictArgs& a, int kv, bool both, cudaStream_t cs) {
    return both ? move_as<V, FOUR, true>(a, kv, cs) : move_as<V, FOUR, false>(a, kv, cs);
}

template <int THREADS>
cudaError_t choose(const EvictArgs& a, cudaStream_t cs) {
    const int smem = (int)(a.acc_ld < HELD ? (a.acc_ld + 7) / 8 * 8 : HELD) * 4;
    if (smem > 36 * 1024) {      // (beside the block's own tables)
        const cudaError_t e = cudaFuncSetAttribute(evict_choose_kernel<THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, HELD * 4);
        if (e != cudaSuccess) return e;
    }
    launch_chained(evict_choose_kernel<THREADS>, dim3(a.G, a.B, a.layers), THREADS, smem, cs, a);
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
    for (int i = 0; i < 2 * layers && B > 0; ++i) {      // (every one is moved within itself, all at the same time)
        void* const p = i < layers ? kpools[i] : vpools[i - layers];
        for (int j = 0; j < i; ++j)
            if (p == (j < layers ? kpools[j] : vpools[j - layers]) || (i < layers && accs[i] == accs[j])) return fail(B200SEQ_ERR_INVALID_ARG, "evict_keys: a pool, or weights, given twice");
    }
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
        // (a slot of up to 8192 weights: eight blocks an SM; more: one or two)
        cudaError_t err = acc_ld <= 8192 ? choose<256>(a, cs) : choose<1024>(a, cs);
        if (err != cudaSuccess) return cuda_status(err, "evict_keys");
        count_launch();
        for (int kv = 0; kv < 2; ++kv) {
            const int size = kv ? V : D;
            if (kv_bits == 4) a.ng[kv] = kv4_groups(size), a.units[kv] = 5;
            else a.units[kv] = wide[kv] ? size / 4 : size;
        }
        const bool both = a.units[0] == a.units[1] && a.ng[0] == a.ng[1] && wide[0] == wide[1];
        for (int kv = 0; kv < (both ? 1 : 2); ++kv) {
            if (kv_bits == 4) err = a.ng[kv] == 4 ? move<uint4, true>(a, kv, both, cs) : a.ng[kv] == 2 ? move<uint2, true>(a, kv, both, cs) : move<uint32_t, true>(a, kv, both, cs);
            else err = wide[kv] ? move<uint4, false>(a, kv, both, cs) : move<uint32_t, false>(a, kv, both, cs);
            if (err != cudaSuccess) return cuda_status(err, "evict_keys");
            count_launch();
        }
    }
    return 0;
}
