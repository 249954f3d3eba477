// One token a row by temperature, top-k, top-p and min-p from a given uniform number.
//
// A token's weight exp((x - max) / T) is held as a whole number of 2^-31, its mass.  Sums of whole numbers are the same in any order, so the kept
// set and the token do not depend on how the row was cut up, and need no sorted running sum: "the shortest run of the largest
// that holds p of the mass" is a threshold c on (logit, lower index first), the least with mass(above c) < p * mass, and top-k is the same with
// counts.  The order of two tokens is that of the 64-bit number (bits of the logit, made to grow with it) : (all ones - index).
#include "common.cuh"

namespace qmoe {
namespace {

constexpr int kThreads = 1024;
constexpr float kOne = 2147483648.f;     // 2^31: the mass of the largest logit's token
constexpr long long kMaxVocab = 1ll << 22;

struct SampleParams {
    const void* logits;
    const float* uniforms;
    const float* temperatures;
    const float* top_ps;
    const float* min_ps;
    const int* top_ks;
    long long* tokens;
    float* log_probs;
    long long rows;
    int vocab, top_k;
    float temperature, top_p, min_p;
};

__device__ __forceinline__ float logit_of(float x) { return isnan(x) ? -INFINITY : x + 0.f; }     // + 0: one zero
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long place_of(float x, int i) { return (unsigned long long)ordered(x) << 32 | (0xffffffffu - (uint32_t)i); }
__device__ __forceinline__ float weight_of(float x, float largest, float inverse) {
    const float apart = x - largest;
    return x == largest ? 1.f : apart == -INFINITY ? 0.f : expf(apart * inverse);
}
__device__ __forceinline__ uint32_t mass_of(float weight) { return __float2uint_rn(weight * kOne); }

// over the block, in every thread
__device__ unsigned long long block_sum(unsigned long long v, unsigned long long* scratch) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
sample_kernel(const __grid_constant__ SampleParams p) {
    chain_begin();
    __shared__ unsigned long long s_scratch[32];
    __shared__ float s_max[32];
    const long long row = blockIdx.x;
    const T* x = (const T*)p.logits + row * p.vocab;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float temperature = p.temperatures ? p.temperatures[row] : p.temperature;
    const float top_p = p.top_ps ? p.top_ps[row] : p.top_p, min_p = fminf(p.min_ps ? p.min_ps[row] : p.min_p, 1.f);
    const bool greedy = !(temperature > 0.f);
    const float inverse = greedy ? 1.f : __fdiv_rn(1.f, temperature);
    const int top_k = greedy ? 1 : p.top_ks ? p.top_ks[row] : p.top_k;

    float largest = -INFINITY;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) largest = fmaxf(largest, logit_of(Act<T>::load(x + i)));
    largest = warp_max(largest);
    if (lane == 0) s_max[warp] = largest;
    __syncthreads();
    largest = warp_max(s_max[lane]);
    if (largest == -INFINITY) {
        if (threadIdx.x == 0) { p.tokens[row] = -1; p.log_probs[row] = -INFINITY; }
        return;
    }
    // mass or number of the tokens in [from, ...) above c
    auto above = [&](unsigned long long c, unsigned long long from, bool count) {
        unsigned long long sum = 0;
        for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
            const float v = logit_of(Act<T>::load(x + i));
            const unsigned long long place = place_of(v, i);
            if (place > c && place >= from) sum += count ? 1u : mass_of(weight_of(v, largest, inverse));
        }
        return block_sum(sum, s_scratch);
    };
    unsigned long long first = 0;        // the least place that is kept
    if (top_k > 0 && top_k < p.vocab)
        for (int bit = 63; bit >= 0; --bit)
            if (above(first | ((1ull << bit) - 1), 0, true) >= (unsigned long long)top_k) first |= 1ull << bit;
    const unsigned long long whole = above(0, 0, false);
    if (top_p < 1.f || isnan(top_p)) {
        const double threshold = (double)top_p * (double)above(0, first, false);
        unsigned long long c = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long before = above(c | ((1ull << bit) - 1), first, false);
            if (!(before == 0 || (double)before < threshold)) c |= 1ull << bit;
        }
        first = c > first ? c : first;
    }
    // a run of neighbouring tokens to a thread
    const int run = (p.vocab + kThreads - 1) / kThreads, begin = min(p.vocab, (int)threadIdx.x * run), end = min(p.vocab, begin + run);
    auto kept = [&](int i) -> uint32_t {
        const float v = logit_of(Act<T>::load(x + i)), weight = weight_of(v, largest, inverse);
        return place_of(v, i) >= first && !(weight < min_p) ? mass_of(weight) : 0u;
    };
    unsigned long long mine = 0;
    for (int i = begin; i < end; ++i) mine += kept(i);
    unsigned long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    __syncthreads();
    if (lane == 31) s_scratch[warp] = upto;
    __syncthreads();
    unsigned long long total = 0;
    for (int w = 0; w < 32; ++w) {
        if (w == warp) upto += total;
        total += s_scratch[w];
    }
    long long target = (long long)((double)p.uniforms[row] * (double)total);
    target = max(0ll, min(target, (long long)total - 1));
    if ((unsigned long long)target >= upto - mine && (unsigned long long)target < upto) {
        unsigned long long sum = upto - mine;
        int i = begin;
        for (; i < end; ++i) {
            sum += kept(i);
            if (sum > (unsigned long long)target) break;
        }
        p.tokens[row] = i;
        const float v = logit_of(Act<T>::load(x + i)), z = v == largest ? 0.f : (v - largest) * inverse;
        p.log_probs[row] = (float)((double)z - log((double)whole / (double)kOne));
    }
}

}  // namespace
}  // namespace qmoe

using namespace qmoe;

extern "C" int qmoe_sample(const qmoe_sample_t* a, uint64_t stream_) {
    if (!a) return fail_arg("sample: argument is null");
    if (a->dtype != QMOE_F32 && a->dtype != QMOE_BF16) return fail_arg("sample: dtype must be QMOE_F32 or QMOE_BF16");
    if (a->rows < 0 || a->vocab <= 0 || a->vocab > kMaxVocab || a->rows > 0x7fffffff) return fail_arg("sample: rows must not be negative, vocab between 1 and %lld", kMaxVocab);
    if (a->top_k < 0 || !(a->top_p > 0) || !(a->min_p >= 0) || !(a->temperature >= 0))
        return fail_arg("sample: top_k, min_p and temperature must not be negative, top_p must be positive");
    if (!a->logits || !a->uniforms || !a->tokens || !a->log_probs) return fail_arg("sample: null buffer address");
    if (a->logits & (a->dtype == QMOE_BF16 ? 1u : 3u) || (a->uniforms | a->temperatures | a->top_ps | a->min_ps | a->top_ks | a->log_probs) & 3u || a->tokens & 7u)
        return fail_arg("sample: misaligned address");
    if (!a->rows) return 0;
    cudaStream_t stream = (cudaStream_t)stream_;
    TimedScope timed(KC_OTHER, stream);
    SampleParams p = {};
    p.logits = (const void*)a->logits; p.uniforms = (const float*)a->uniforms;
    p.temperatures = (const float*)a->temperatures; p.top_ps = (const float*)a->top_ps; p.min_ps = (const float*)a->min_ps; p.top_ks = (const int*)a->top_ks;
    p.tokens = (long long*)a->tokens; p.log_probs = (float*)a->log_probs;
    p.rows = a->rows; p.vocab = (int)a->vocab; p.top_k = a->top_k; p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p;
    if (a->dtype == QMOE_BF16) chained(sample_kernel<__nv_bfloat16>, (unsigned)a->rows, kThreads, 0, stream, p);
    else chained(sample_kernel<float>, (unsigned)a->rows, kThreads, 0, stream, p);
    QMOE_LAUNCH_CHECK("sample_kernel");
    return 0;
}
