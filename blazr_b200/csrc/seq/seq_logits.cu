// seq_logits.cu -- what a request's sampling rules make of its logits, in one pass over the row: penalties for repeated tokens, biases, temperature, grammar mask.
//
// A block has a slice of one row's vocabulary.  It counts the row's history into a table in shared memory (only the tokens of its slice; whole numbers, so the order of
// the additions does not matter), then reads, changes and writes its logits once.  The floor is the logits' bytes, 8 a token; a block's time is a
// chain of loads (bounds, history, counts, biases), the history is read by every slice, from L2.  64 rows of 128256: 16 us without rules (4.1 TB/s), 26 with histories of up to
// 4000 tokens, 30 with 300 biases and a mask too; one row of 32000 with 500 tokens 2.4.
#include "seq_common.cuh"

namespace b200seq {

namespace {

constexpr int ERR_TOKEN = 16;            // error flag: a token id outside the vocabulary
constexpr uint32_t SEEN = 0x80000000u;   // in the table: the token stands in the prompt

struct LogitArgs {
    const float* x;
    float* out;
    int64_t ldx, ldo;
    int V;
    const float* rules;                        // [R][4]: repetition, presence, frequency, temperature
    const int32_t *hist, *hist_start, *hist_prompt;
    const int32_t *bias_start, *bias_ids;
    int nhist, nbias;
    const float* bias_vals;
    const uint32_t* mask;                      // [R][mask_ld]: bit v % 32 of word v / 32
    int64_t mask_ld;
    int vec;
    int* err;
};

// grid (slices of 4 * ITEMS * THREADS tokens, rows).  Dynamic shared memory: the counts and, with biases, the number of the entry that holds for a token.
// What a block needs first of memory is asked for before its tables are cleared: a chain of loads, not the bytes, is what a block's time is.
template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 2 : 1) process_logits_kernel(const __grid_constant__ LogitArgs a) {
    chain_enter();
    constexpr int S = 4 * ITEMS * THREADS;
    extern __shared__ __align__(16) uint32_t table[];
    uint32_t* entry = table + S;
    const int row = blockIdx.y, v0 = blockIdx.x * S, n = min(S, a.V - v0);
    const float4 rule = ld4(a.rules + 4 * (int64_t)row);   // repetition, presence, frequency, temperature
    int h0 = 0, h1 = 0, prompt = 0, b0 = 0, b1 = 0;
    if (a.hist) h0 = a.hist_start[row], h1 = a.hist_start[row + 1], prompt = a.hist_prompt[row];
    if (a.bias_ids) b0 = a.bias_start[row], b1 = a.bias_start[row + 1];
    const float* x = a.x + row * a.ldx + v0;
    float4 v[ITEMS];
    uint32_t bits[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = 4 * (k * THREADS + threadIdx.x);
        if (a.vec && i + 3 < n) v[k] = ld4(x + i);
        else v[k] = make_float4(i < n ? x[i] : 0.f, i + 1 < n ? x[i + 1] : 0.f, i + 2 < n ? x[i + 2] : 0.f, i + 3 < n ? x[i + 3] : 0.f);
        bits[k] = a.mask && i < n ? a.mask[row * a.mask_ld + ((v0 + i) >> 5)] >> ((v0 + i) & 31) : 0xFu;
    }
    // a row's list that is not one: the row has none
    bool odd = h0 < 0 || h0 > h1 || h1 > a.nhist || b0 < 0 || b0 > b1 || b1 > a.nbias;
    if (odd) h0 = h1 = b0 = b1 = 0;
    prompt += h0;
    const bool biased = b1 > b0;
    for (int i = threadIdx.x; i < (biased ? 2 * S : S) / 4; i += THREADS) reinterpret_cast<uint4*>(table)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
#pragma unroll 4
    for (int i = h0 + (int)threadIdx.x; i < h1; i += THREADS) {
        const int id = a.hist[i];
        if ((unsigned)(id - v0) < (unsigned)n) {
            if (i < prompt) atomicOr(table + (id - v0), SEEN);
            else atomicAdd(table + (id - v0), 1u);
        }
        odd |= (unsigned)id >= (unsigned)a.V;
    }
    for (int i = b0 + (int)threadIdx.x; i < b1; i += THREADS) {
        const int id = a.bias_ids[i];
        if ((unsigned)(id - v0) < (unsigned)n) atomicMax(entry + (id - v0), (uint32_t)(i - b0 + 1));
        odd |= (unsigned)id >= (unsigned)a.V;
    }
    if (odd && blockIdx.x == 0) atomicOr(a.err, ERR_TOKEN);
    __syncthreads();
    float* out = a.out + row * a.ldo + v0;
    const float heat = rule.w != 0.f ? rule.w : 1.f;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = 4 * (k * THREADS + threadIdx.x);
        if (i >= n) continue;
        const uint4 cnt = *reinterpret_cast<const uint4*>(table + i);
        float y[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
        if (cnt.x | cnt.y | cnt.z | cnt.w) {
            const uint32_t cs[4] = {cnt.x, cnt.y, cnt.z, cnt.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!cs[j]) continue;
                y[j] = y[j] > 0.f ? y[j] / rule.x : y[j] * rule.x;
                const uint32_t times = cs[j] & ~SEEN;
                if (times) y[j] = y[j] - (float)times * rule.z - rule.y;
            }
        }
        if (biased) {
            const uint4 at = *reinterpret_cast<const uint4*>(entry + i);
            if (at.x) y[0] += a.bias_vals[b0 + (int)at.x - 1];
            if (at.y) y[1] += a.bias_vals[b0 + (int)at.y - 1];
            if (at.z) y[2] += a.bias_vals[b0 + (int)at.z - 1];
            if (at.w) y[3] += a.bias_vals[b0 + (int)at.w - 1];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = (bits[k] >> j) & 1u ? y[j] / heat : -INFINITY;
        if (a.vec && i + 3 < n) *reinterpret_cast<float4*>(out + i) = make_float4(y[0], y[1], y[2], y[3]);
        else
            for (int j = 0; j < 4 && i + j < n; ++j) out[i + j] = y[j];
    }
}

template <int THREADS, int ITEMS>
cudaError_t launch(const LogitArgs& a, int R, cudaStream_t cs) {
    constexpr int S = 4 * ITEMS * THREADS;
    const size_t smem = (size_t)S * 4 * (a.bias_ids ? 2 : 1);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(process_logits_kernel<THREADS, ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * S * 4);
        if (e != cudaSuccess) return e;
    }
    launch_chained(process_logits_kernel<THREADS, ITEMS>, dim3((a.V + S - 1) / S, R), THREADS, smem, cs, a);
    return cudaGetLastError();
}

}  // namespace

}  // namespace b200seq

using namespace b200seq;

extern "C" int b200seq_process_logits(const float* x, int64_t ldx, int R, int V, const float* rules, const int32_t* hist, int nhist, const int32_t* hist_start,
                                      const int32_t* hist_prompt, const int32_t* bias_start, const int32_t* bias_ids, const float* bias_vals, int nbias, const uint32_t* mask,
                                      int64_t mask_ld, float* out, int64_t ldo, void* stream) {
    if (R < 0 || V < 1 || (R > 0 && (!x || !out || !rules))) return fail(B200SEQ_ERR_INVALID_ARG, "process_logits: bad sizes or null arrays");
    if (nhist < 0 || nbias < 0) return fail(B200SEQ_ERR_INVALID_ARG, "process_logits: negative lengths");
    if ((hist != nullptr) != (hist_start != nullptr) || (hist != nullptr) != (hist_prompt != nullptr)) return fail(B200SEQ_ERR_INVALID_ARG, "process_logits: a history has ids, row starts and prompt lengths");
    if ((bias_ids != nullptr) != (bias_start != nullptr) || (bias_ids != nullptr) != (bias_vals != nullptr)) return fail(B200SEQ_ERR_INVALID_ARG, "process_logits: biases have ids, values and row starts");
    if (R > 65535) return fail(B200SEQ_ERR_UNSUPPORTED, "process_logits: up to 65535 rows");
    if (R > 1 && (ldx < V || ldo < V || (mask && mask_ld < (V + 31) / 32))) return fail(B200SEQ_ERR_INVALID_ARG, "process_logits: row strides below a row's length");
    if (reinterpret_cast<uintptr_t>(rules) & 15) return fail(B200SEQ_ERR_INVALID_ARG, "process_logits: rules start on a 16-byte boundary");
    if (R == 0) return 0;
    const LogitArgs a{x, out, ldx, ldo, V, rules, hist, hist_start, hist_prompt, bias_start, bias_ids, nhist, nbias, bias_vals, mask, mask_ld,
                      ((ldx | ldo) & 3) == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15) == 0, error_flag_dev()};
    // Every slice reads the row's whole history: slices of 8192 tokens where they fill the GPU, of 1024 otherwise.
    const cudaError_t e = (int64_t)R * ((V + 8191) / 8192) >= 2 * 148 ? launch<1024, 2>(a, R, (cudaStream_t)stream) : launch<256, 1>(a, R, (cudaStream_t)stream);
    if (e != cudaSuccess) return cuda_status(e, "process_logits");
    count_launch();
    return 0;
}
