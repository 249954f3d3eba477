// Causal attention within each of many sequences that lie behind one another in one matrix of rows, grouped key/value heads of width 64 or
// 128, bf16, forward and backward, on the tcgen05 tensor cores:
//     out[t, h, :] = sum_{s <= t, same sequence} softmax_s(scale q[t, h, :] . k[s, g(h), :]) v[s, g(h), :],   g(h) = h / (heads / kv_heads)
// The division of work is that of attention.cu (which says what its parts are): a CTA to 128 queries of a head, or to 128 keys of a key/value head, warp 0 at
// the TMA unit, warp 1 at the tensor cores, the row warps with a lane of tensor memory to a thread; probabilities never pass through shared memory.
//
// What is different:
//   * Blocks of 128 positions are counted from each sequence's own start.  The host lists them (start row, length, block), those with the most blocks
//     to walk first, so the grid has no CTA without work.  A block's tile may reach into the next sequence: its keys lie behind every query that counts
//     and are masked like any later key, its queries are not stored.  What lies behind the last sequence is not read.
//   * A masked position has a probability of 0, and 0 times a value that is no number is none.  Looking for such values in every tile would cost
//     every block, so a row that comes out with one is formed once more, from its own sequence's visible positions alone and without tensor cores: the same
//     result if the value was one that the row sees, and the right one if it was not.
//   * Forward and dq walk key blocks of 64 positions, so that S has two buffers in the 256 columns of a CTA and two CTAs stay on an SM: the scores of the next block are
//     formed while the rows have this one's.  P lies over the S that it came from, and so does dS (heads of 64); with heads of 128 dq has one S, and dS lies over dP.
//     dk, dv has 128 x 128 blocks, 16 row warps and one CTA an SM; with heads of 128 its accumulators leave one buffer each for S and dP.
// What bounds it: the row warps' chain from a block's scores to its probabilities (the exponential unit is busy for 39 % of the forward, the tensor cores for 21 to 36 %, an
// instruction issues in 40 to 45 % of the cycles: 17 documents of up to 2048, 16 heads of 64), and with short documents the CTAs' starts and ends.  Forward and
// backward of 4 x 4096 tokens, 16 query heads of 64 in 4 groups: 737 us, 653 TFLOP/s; 8 heads of 128: 599 us, 803 TFLOP/s.
// No atomics, every sum in a fixed order.  Every wait is bounded; on expiry the CTA records a code in the library's status word and leaves.
#include "common.cuh"
#include "attention_ptx.cuh"

namespace qmoe {
namespace {

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// A value that all lanes have, known to the compiler as one: loop counters, addresses and descriptors that follow from it stay in uniform registers,
// where the tensor-core instructions want them.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
// 2^x of two numbers on the FMA units: x = n + f with n whole and |f| <= 1/2 (an addition of 1.5 * 2^23 rounds to n and leaves it in the low bits), a
// polynomial of degree 5 in f that is off by 2^-22 at most (least largest relative error over [-1/2, 1/2], fitted for this), times 2^n from its exponent's
// bits.  Below -126.5 zero, NaN stays NaN; for x up to 127.
__device__ __forceinline__ float at_least(float x, float least) {      // unlike fmaxf a NaN stays one
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(least));
    return y;
}
__device__ __forceinline__ void exp2_two(uint64_t x, float& p0, float& p1) {
    const auto both = [](float v) { return pair2(v, v); };
    float x0, x1, t0, t1;
    unpair2(x, x0, x1);
    x = pair2(at_least(x0, -127.f), at_least(x1, -127.f));
    const uint64_t t = add2(x, both(12583039.f));                        // n + 127 in the low bits
    const uint64_t f = fma2(add2(t, both(-12583039.f)), both(-1.f), x);
    uint64_t p = fma2(f, both(0.0013276472f), both(0.0096755419f));
    p = fma2(p, f, both(0.0555071309f));
    p = fma2(p, f, both(0.2402212024f));
    p = fma2(p, f, both(0.6931469440f));
    p = fma2(p, f, both(1.0000001192f));
    unpair2(t, t0, t1);
    unpair2(mul2(p, pair2(__uint_as_float(__float_as_uint(t0) << 23), __uint_as_float(__float_as_uint(t1) << 23))), p0, p1);
}
// Forward and dq: of as many pairs of probabilities one is formed there, beside the exponential unit, which is the busiest part of the forward.  4 x 4096 tokens, 16
// heads of 64, with none, one of 8, 4, 3 and 2: forward 240, 230, 233, 236 and 264 us, dq 443, 417, 416, 414 and 433 thousand cycles; 8 heads of 128: forward 157,
// 154, 153, 158 and 171 us, dq 331, 330, 332, 331 and 340 thousand cycles.
constexpr int ON_FMA = 8;

struct QuickWait {
    Wait slow;
    __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const { return slow(bar, parity); }
    __device__ __forceinline__ bool all(uint32_t bar, uint32_t parity) const {
        if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
        return slow.all(bar, parity);
    }
};

constexpr int BLOCK = 128;                      // query rows of a CTA = key positions of a block
constexpr int THREADS = 192;                    // forward, dq: TMA warp, MMA warp, four row warps
constexpr int DKV_PARTS = 4, DKV_THREADS = 64 + 128 * DKV_PARTS;

struct alignas(64) PackedParams {
    CUtensorMap map_q, map_k, map_v, map_do;    // [rows][heads * D] bf16 in boxes of 64 columns x 128 rows (k, v of the dq kernel: 64 rows)
    const int4* items;                          // {first row of the sequence, its length, block, -}
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    const __nv_bfloat16* out_in;                // backward: the forward's output
    const __nv_bfloat16* grad_out;
    __nv_bfloat16* out;                         // forward: out; dq: dq; dk, dv: dk
    __nv_bfloat16* out2;                        // dk, dv: dv
    float* lse;                                 // [rows, heads]
    float* delta;                               // [rows, heads]  sum_j grad_out * out
    int* status;
    long long q_pitch, k_pitch, v_pitch;
    float scale;
    int heads, kv_heads;
    int split, shared, jobs;                    // dk, dv: CTAs of a cluster, lists that are a whole cluster's, lists
};

__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float sum) {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sum = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), sum);
        sum = fmaf(__uint_as_float(x[i] & 0xffff0000u), __uint_as_float(y[i] & 0xffff0000u), sum);
    }
    return sum;
}
template <int D> __device__ __forceinline__ float dot_rows(const __nv_bfloat16* a, const __nv_bfloat16* b) {
    float sum = 0.f;
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) sum = dot8(reinterpret_cast<const uint4*>(a)[c], reinterpret_cast<const uint4*>(b)[c], sum);
    return sum;
}
__device__ __forceinline__ void add_scaled8(const uint4& a, float by, float* sum) {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sum[2 * i] = fmaf(by, __uint_as_float(x[i] << 16), sum[2 * i]);
        sum[2 * i + 1] = fmaf(by, __uint_as_float(x[i] & 0xffff0000u), sum[2 * i + 1]);
    }
}
// Rows that came out with a value that is no number, once more from the positions that they see (64 columns at a time, from `column` on).
template <int D>
__device__ __noinline__ void forward_again(const PackedParams& p, int start, int tq, int h, int g, float base, float inverse) {
    const __nv_bfloat16* q = p.q + (start + (long long)tq) * p.q_pitch + h * D;
    for (int column = 0; column < D; column += 32) {
        float o[32] = {};
        for (int s = 0; s <= tq; ++s) {
            const long long row = start + (long long)s;
            const float weight = exp2_fast((dot_rows<D>(q, p.k + row * p.k_pitch + g * D) - base) * (p.scale * LOG2E));
            const uint4* v = reinterpret_cast<const uint4*>(p.v + row * p.v_pitch + g * D + column);
#pragma unroll
            for (int c = 0; c < 4; ++c) add_scaled8(v[c], weight, o + 8 * c);
        }
        store_row32(reinterpret_cast<uint4*>(p.out + ((start + (long long)tq) * p.heads + h) * D + column), reinterpret_cast<const uint32_t*>(o), inverse);
    }
}
template <int D>
__device__ __noinline__ void dq_again(const PackedParams& p, int start, int tq, int h, int g, float lse2, float delta) {
    const long long at = (start + (long long)tq) * p.heads + h;
    const __nv_bfloat16 *q = p.q + (start + (long long)tq) * p.q_pitch + h * D, *grad = p.grad_out + at * D;
    for (int column = 0; column < D; column += 32) {
        float dq[32] = {};
        for (int s = 0; s <= tq; ++s) {
            const long long row = start + (long long)s;
            const __nv_bfloat16* k = p.k + row * p.k_pitch + g * D;
            const float weight = exp2_fast(fmaf(dot_rows<D>(q, k), p.scale * LOG2E, -lse2));
            const float ds = weight * (dot_rows<D>(grad, p.v + row * p.v_pitch + g * D) - delta);
#pragma unroll
            for (int c = 0; c < 4; ++c) add_scaled8(reinterpret_cast<const uint4*>(k + column)[c], ds, dq + 8 * c);
        }
        store_row32(reinterpret_cast<uint4*>(p.out + at * D + column), reinterpret_cast<const uint32_t*>(dq), p.scale);
    }
}
// 32 columns of one key's dv (chunks 0 .. D / 32 - 1) or dk (those behind), over `n` iterations from (first_head, first_i) on
template <int D>
__device__ __noinline__ void dkv_again(const PackedParams& p, int start, int length, int s, int g, int j, int first_head, int first_i, int n, int chunk, uint32_t* sums) {
    const int blocks = (length + BLOCK - 1) / BLOCK, group = p.heads / p.kv_heads, column = chunk % (D / 32) * 32;
    const __nv_bfloat16 *k = p.k + (start + (long long)s) * p.k_pitch + g * D, *v = p.v + (start + (long long)s) * p.v_pitch + g * D;
    float sum[32] = {};
    int head = first_head, i = first_i;
    for (int it = 0; it < n; ++it) {
        const int h = g * group + head;
        for (int t = max(s, i * BLOCK); t < min(length, (i + 1) * BLOCK); ++t) {
            const long long at = (start + (long long)t) * p.heads + h;
            const __nv_bfloat16 *q = p.q + (start + (long long)t) * p.q_pitch + h * D, *grad = p.grad_out + at * D;
            float weight = exp2_fast(fmaf(dot_rows<D>(q, k), p.scale * LOG2E, -p.lse[at] * LOG2E));
            if (chunk >= D / 32) weight *= dot_rows<D>(grad, v) - p.delta[at];
            const uint4* from = reinterpret_cast<const uint4*>((chunk >= D / 32 ? q : grad) + column);
#pragma unroll
            for (int c = 0; c < 4; ++c) add_scaled8(from[c], weight, sum + 8 * c);
        }
        if (++i == blocks) { i = j; ++head; }
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) sums[e] = __float_as_uint(sum[e]);
}
// 0 while all 32 are finite numbers, else not a number
__device__ __forceinline__ float oddness(const uint32_t* r) {
    float z = 0.f;
#pragma unroll
    for (int e = 0; e < 32; ++e) z = fmaf(__uint_as_float(r[e]), 0.f, z);
    return z;
}

__device__ __forceinline__ void load_tile(const CUtensorMap* map, uint32_t dst, uint32_t bar, int column, int row, int width, int part_bytes) {
    for (int c = 0; c < width; c += 64) tma_load_2d(map, dst + c / 64 * part_bytes, bar, column + c, row);
}
// where the contraction elements [16 kk, 16 kk + 16) of a K-major tile lie, whose parts of 64 columns are `part` bytes apart
template <int PART> __device__ __forceinline__ constexpr uint32_t k_major(int kk) { return (uint32_t)(kk / 4 * PART + kk % 4 * 32); }

__device__ __forceinline__ void allocate(uint32_t* base, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void release(uint32_t tmem, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

// The CTA's entry of the table, by one warp beside the set-up of the others.  The kernel before this one may still be writing the table: behind the wait.
__device__ __forceinline__ void fetch_item(const PackedParams& p, int which, int* to) {
    chain_wait();
    if ((threadIdx.x & 31) == 0) {
        const int4 item = p.items[which];
        to[0] = item.x; to[1] = item.y; to[2] = item.z;
    }
}

// ------------------------------------------------------------------------------------------------
// forward: a CTA to 128 queries of a head, key blocks of 64 positions.  S has two buffers, P lies over the S that it came from: the next
// scores are formed while the rows have this block's, and a row waits for nothing but them.
// ------------------------------------------------------------------------------------------------
constexpr int KEYS = 64;                               // positions of a key block (forward, dq)
template <int D> struct Forward {
    static constexpr int PART = BLOCK * 128, TILE = D / 64 * PART;             // Q: 64 columns of it, the tile
    static constexpr int KV_PART = KEYS * 128, KV_TILE = D / 64 * KV_PART;     // K, V
    static constexpr int STAGES = D == 64 ? 3 : 2;                             // of K, of V
    static constexpr int TILES = TILE + 2 * STAGES * KV_TILE;
    enum { Q_FULL = 0, K_FULL = 1, K_EMPTY = K_FULL + STAGES, V_FULL = K_EMPTY + STAGES, V_EMPTY = V_FULL + STAGES, S_FULL = V_EMPTY + STAGES, P_FULL = S_FULL + 2, O_DONE = P_FULL + 2, O_LAST, BARS };
    // (P_FULL is two barriers, by the parity of the block: a warp may have the next block's scores, and be done with them, before another one is done with this block's)
    static constexpr int SMEM = TILES + 8 * BARS + 24;
};

template <int D>
__global__ void __launch_bounds__(THREADS, 2)
packed_forward_kernel(const __grid_constant__ PackedParams p) {
    using C = Forward<D>;
    constexpr int TILE = C::TILE, PART = C::PART, KV_TILE = C::KV_TILE, KV_PART = C::KV_PART, STAGES = C::STAGES;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem_raw);
    const uint32_t q_tile = base, k_tile = base + TILE, v_tile = k_tile + STAGES * KV_TILE, bars = base + C::TILES;
    auto bar = [&](int which) { return bars + 8u * which; };
    uint32_t& s_tmem_base = *reinterpret_cast<uint32_t*>(smem_raw + C::TILES + 8 * C::BARS);
    volatile int& s_abort = *reinterpret_cast<volatile int*>(smem_raw + C::TILES + 8 * C::BARS + 4);
    int* s_item = reinterpret_cast<int*>(smem_raw + C::TILES + 8 * C::BARS + 8);
    if (base & 1023u) {   // the operand tiles need the alignment the declaration asks for
        chain_wait();
        if (threadIdx.x == 0) atomicExch(p.status, STATUS_ATTENTION_WAIT + 1);
        return;
    }
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int w = 0; w < C::BARS; ++w) mbar_init(bar(w), w == C::P_FULL || w == C::P_FULL + 1 ? 4 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&p.map_q); prefetch_map(&p.map_k); prefetch_map(&p.map_v);
    }
    if (warp == 1) allocate(&s_tmem_base, 256);
    if (warp == 2) fetch_item(p, blockIdx.x / p.heads, s_item);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    chain_wait();
    chain_next();      // the tensor memory is this block's
    const int start = uniform(s_item[0]), length = uniform(s_item[1]), i = uniform(s_item[2]);
    const int h = (int)(blockIdx.x % p.heads), g = h / (p.heads / p.kv_heads);
    // key blocks that hold a position <= the last query of this block that there is
    const int n = (min(length, (i + 1) * BLOCK) + KEYS - 1) / KEYS;
    const uint32_t tmem = s_tmem_base, tmem_o = tmem + 2 * KEYS;
    const QuickWait wait{{&s_abort, p.status}};

    if (warp == 0) {
        if (lane == 0) {
            mbar_expect_tx(bar(C::Q_FULL), TILE);
            load_tile(&p.map_q, q_tile, bar(C::Q_FULL), h * D, start + i * BLOCK, D, PART);
            int st = 0;
            uint32_t parity = 1;
            for (int j = 0; j < n && !s_abort; ++j) {
                if (!wait(bar(C::K_EMPTY + st), parity)) break;
                mbar_expect_tx(bar(C::K_FULL + st), KV_TILE);
                load_tile(&p.map_k, k_tile + st * KV_TILE, bar(C::K_FULL + st), g * D, start + j * KEYS, D, KV_PART);
                if (!wait(bar(C::V_EMPTY + st), parity)) break;
                mbar_expect_tx(bar(C::V_FULL + st), KV_TILE);
                load_tile(&p.map_v, v_tile + st * KV_TILE, bar(C::V_FULL + st), g * D, start + j * KEYS, D, KV_PART);
                if (++st == STAGES) { st = 0; parity ^= 1u; }
            }
        }
    } else if (warp == 1) {
        // One lane, elected once, walks the blocks by itself, with the descriptors formed once: the warp's votes on every wait, an election for every product and a
        // descriptor for every instruction cost 2 to 6 % of the time of each of the three kernels (4 x 4096 tokens: dk, dv of 64 528 to 496 thousand cycles).
        if (elect_one()) {
            constexpr uint32_t idesc_s = make_idesc<false, false, 128>(KEYS), idesc_o = make_idesc<false, true, 128>(D);
            const uint64_t q_desc = make_desc(q_tile, 16, 1024), k_desc = make_desc(k_tile, 16, 1024), v_desc = make_desc(v_tile, KV_PART, 1024);
            auto scores = [&](int j) {      // S = Q K^T of key block j into its buffer
                const int st = j % STAGES;
                if (!wait(bar(C::K_FULL + st), (uint32_t)(j / STAGES) & 1u)) return false;
                tc_fence_after();
                const uint64_t k_of = k_desc + (uint64_t)(st * (KV_TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma_bf16(tmem + (uint32_t)(j & 1) * KEYS, q_desc + (k_major<PART>(kk) >> 4), k_of + (k_major<KV_PART>(kk) >> 4), idesc_s, kk ? 1u : 0u);
                umma_commit(bar(C::S_FULL + (j & 1)));
                umma_commit(bar(C::K_EMPTY + st));
                return true;
            };
            bool ok = wait(bar(C::Q_FULL), 0) && scores(0);
            for (int j = 0; ok && j < n; ++j) {
                const int st = j % STAGES;
                // the next scores into the other buffer, once the product that reads the P of block j - 1 there is done
                if (j > 0) ok = wait(bar(C::O_DONE), (uint32_t)(j - 1) & 1u);
                if (ok && j + 1 < n) ok = scores(j + 1);
                if (ok) ok = wait(bar(C::V_FULL + st), (uint32_t)(j / STAGES) & 1u);
                if (ok) ok = wait(bar(C::P_FULL + (j & 1)), (uint32_t)(j >> 1) & 1u);
                if (!ok) break;
                tc_fence_after();
                // O += P V: P from tensor memory, V as it lies in memory (rows = key positions) the MN-major operand
                const uint64_t v_of = v_desc + (uint64_t)(st * (KV_TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < KEYS / 16; ++kk)
                    umma_bf16_ts(tmem_o, tmem + (uint32_t)(j & 1) * KEYS + kk * 8, v_of + (uint64_t)(kk * (2048 >> 4)), idesc_o, (j | kk) ? 1u : 0u);
                umma_commit(bar(C::V_EMPTY + st));
                umma_commit(bar(j + 1 < n ? C::O_DONE : C::O_LAST));
            }
            // the last commit has arrived before this CTA's shared memory can go to another one
            if (ok) wait(bar(C::O_LAST), 0);
        }
        __syncwarp();
    } else {
        const int quad = warp & 3, row = quad * 32 + lane, tq = i * BLOCK + row;
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const float scale2 = p.scale * LOG2E;                // in the exponent of 2
        const uint64_t scale_pair = pair2(scale2, scale2);
        // What is subtracted from scores: the largest so far (0 while all are -infinity), so that a row's largest probability is an exact 1 in bf16.  A base that may stay
        // up to 2^8 below it leaves O alone in most blocks (forward, 4 x 4096 tokens, 16 heads of 64: 211 us for 230; 8 of 128: 133 for 154), but then that
        // probability is rounded too: out 2.13e-3 instead of 2.06e-3 from the exact result for operands of standard deviation 1, 2.08e-3 instead of 1.74e-3 for 2.
        float from = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; ok && j < n; ++j) {
            const uint32_t tmem_s = tmem + (uint32_t)(j & 1) * KEYS + lane_base;
            const int first = j * KEYS - i * BLOCK;                      // first key position of the block, from the CTA's first query
            ok = wait.all(bar(C::S_FULL + (j & 1)), (uint32_t)(j >> 1) & 1u);
            if (!ok) break;
            tc_fence_after();
            uint32_t s[KEYS];
            tmem_ld32(tmem_s, s);
            tmem_ld32(tmem_s + 32, s + 32);
            tmem_ld_wait();
            if (first + KEYS - 1 > quad * 32) {                          // some row of this warp may not see some of these columns
#pragma unroll
                for (int c = 0; c < KEYS; ++c)
                    if (first + c > row) s[c] = 0xff800000u;             // -inf
            }
            float peak4[4] = {__uint_as_float(s[0]), __uint_as_float(s[1]), __uint_as_float(s[2]), __uint_as_float(s[3])};
#pragma unroll
            for (int c = 4; c < KEYS; c += 2) peak4[(c >> 1) & 3] = max3(peak4[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
            const float peak = fmaxf(max3(peak4[0], peak4[1], peak4[2]), peak4[3]);
            float alpha = 1.f;
            if (peak > from) {
                alpha = exp2_fast((from - peak) * scale2);
                from = peak;
                l *= alpha;
            }
            const float against = from == -INFINITY ? 0.f : from;
            // (subtract, then multiply: a single fma would leave the base rounded, attention.cu)
            const uint64_t minus = pair2(-against, -against);
            uint64_t total2[2] = {0, 0};
            uint32_t packed[KEYS / 2];
#pragma unroll
            for (int c = 0; c < KEYS; c += 2) {
                const uint64_t x = mul2(add2(pair2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), minus), scale_pair);
                float p0, p1;
                if ((c >> 1) % ON_FMA == ON_FMA - 1) {
                    exp2_two(x, p0, p1);
                } else {
                    unpair2(x, p0, p1);
                    p0 = exp2_fast(p0);
                    p1 = exp2_fast(p1);
                }
                total2[(c >> 1) & 1] = add2(total2[(c >> 1) & 1], pair2(p0, p1));
                packed[c >> 1] = pack2(p0, p1);
            }
            if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                ok = wait.all(bar(C::O_DONE), (uint32_t)(j - 1) & 1u);           // O is whole (this block's scores came after the product of block j - 2)
                if (!ok) break;
                tc_fence_after();
                const uint64_t alpha_pair = pair2(alpha, alpha);
                constexpr int AT_ONCE = D == 64 ? 64 : 32;       // (64 of heads of 128 spill: forward 148 us to 156 at 4 x 4096; 32 of heads of 64: 215 to 222)
#pragma unroll
                for (int c = 0; c < D; c += AT_ONCE) {
                    uint32_t o[AT_ONCE];
#pragma unroll
                    for (int e = 0; e < AT_ONCE; e += 32) tmem_ld32(tmem_o + lane_base + c + e, o + e);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < AT_ONCE; e += 2) {
                        float o0, o1;
                        unpair2(mul2(pair2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), alpha_pair), o0, o1);
                        o[e] = __float_as_uint(o0);
                        o[e + 1] = __float_as_uint(o1);
                    }
#pragma unroll
                    for (int e = 0; e < AT_ONCE; e += 32) tmem_st32(tmem_o + lane_base + c + e, o + e);
                }
            }
            tmem_st32(tmem_s, packed);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::P_FULL + (j & 1)));
            float t0, t1;
            unpair2(add2(total2[0], total2[1]), t0, t1);
            l += t0 + t1;
        }
        // (a barrier of its own: a row has not waited for every product, and a parity tells two neighbouring phases apart, no more)
        if (ok) ok = wait.all(bar(C::O_LAST), 0);
        if (ok) {
            tc_fence_after();
            const bool live = tq < length;
            const long long at = (start + (long long)tq) * p.heads + h;
            const float inverse = 1.f / l;
            float odd = 0.f;
            uint4* dst = reinterpret_cast<uint4*>(p.out + at * D);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(tmem_o + lane_base + c * 32, o);
                tmem_ld_wait();
                odd += oddness(o);
                if (live) store_row32(dst + c * 4, o, inverse);
            }
            if (live) {
                p.lse[at] = from * p.scale + __logf(l);
                if (odd != 0.f && l == l) forward_again<D>(p, start, tq, h, g, from, inverse);
            }
        }
    }
    linger_after_abort(&s_abort);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        release(tmem, 256);
    }
}

// ------------------------------------------------------------------------------------------------
// backward, part 1: dq (and delta), a CTA to 128 queries of a head, key blocks of 64 positions
// ------------------------------------------------------------------------------------------------
template <int D> struct DQ {
    static constexpr int PART = BLOCK * 128, TILE = D / 64 * PART;             // Q, dO
    static constexpr int KV_PART = KEYS * 128, KV_TILE = D / 64 * KV_PART;    // K, V
    static constexpr int K_STAGES = D == 64 ? 3 : 2, V_STAGES = D == 64 ? 3 : 1;
    static constexpr int BUFFERS = D == 64 ? 2 : 1;                            // of S; with two dS lies over S, with one over dP
    static constexpr int TILES = 2 * TILE + (K_STAGES + V_STAGES) * KV_TILE;
    enum { Q_FULL = 0, K_FULL = 1, K_EMPTY = K_FULL + K_STAGES, V_FULL = K_EMPTY + K_STAGES, V_EMPTY = V_FULL + V_STAGES, S_FULL = V_EMPTY + V_STAGES,
           S_TAKEN = S_FULL + 2, DP_FULL, DS_FULL, DQ_DONE, BARS };
    static constexpr int SMEM = TILES + 8 * BARS + 24;
};

template <int D>
__global__ void __launch_bounds__(THREADS, 2)
packed_dq_kernel(const __grid_constant__ PackedParams p) {
    using C = DQ<D>;
    constexpr int TILE = C::TILE, PART = C::PART, KV_TILE = C::KV_TILE, KV_PART = C::KV_PART;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem_raw);
    const uint32_t q_tile = base, do_tile = base + TILE, k_tile = do_tile + TILE, v_tile = k_tile + C::K_STAGES * KV_TILE, bars = base + C::TILES;
    auto bar = [&](int which) { return bars + 8u * which; };
    uint32_t& s_tmem_base = *reinterpret_cast<uint32_t*>(smem_raw + C::TILES + 8 * C::BARS);
    volatile int& s_abort = *reinterpret_cast<volatile int*>(smem_raw + C::TILES + 8 * C::BARS + 4);
    int* s_item = reinterpret_cast<int*>(smem_raw + C::TILES + 8 * C::BARS + 8);
    if (base & 1023u) {
        chain_wait();
        if (threadIdx.x == 0) atomicExch(p.status, STATUS_ATTENTION_WAIT + 1);
        return;
    }
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int w = 0; w < C::BARS; ++w) mbar_init(bar(w), w == C::DS_FULL || w == C::S_TAKEN ? 4 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&p.map_q); prefetch_map(&p.map_k); prefetch_map(&p.map_v); prefetch_map(&p.map_do);
    }
    if (warp == 1) allocate(&s_tmem_base, 256);
    if (warp == 2) fetch_item(p, blockIdx.x / p.heads, s_item);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    chain_wait();
    chain_next();      // the tensor memory is this block's
    const int start = uniform(s_item[0]), length = uniform(s_item[1]), i = uniform(s_item[2]);
    const int h = (int)(blockIdx.x % p.heads), g = h / (p.heads / p.kv_heads);
    // key blocks that hold a position <= the last query of this block that there is
    const int n = (min(length, (i + 1) * BLOCK) + KEYS - 1) / KEYS;
    const uint32_t tmem = s_tmem_base;
    // S of block j in columns 64 (j % BUFFERS) ..; the rows put dS (bf16 pairs) back over the S or the dP that they read
    const uint32_t tmem_dp = tmem + C::BUFFERS * KEYS, tmem_dq = tmem_dp + KEYS;
    const QuickWait wait{{&s_abort, p.status}};

    if (warp == 0) {
        if (lane == 0) {
            mbar_expect_tx(bar(C::Q_FULL), 2 * TILE);
            load_tile(&p.map_q, q_tile, bar(C::Q_FULL), h * D, start + i * BLOCK, D, PART);
            load_tile(&p.map_do, do_tile, bar(C::Q_FULL), h * D, start + i * BLOCK, D, PART);
            for (int j = 0; j < n && !s_abort; ++j) {
                const int ks = j % C::K_STAGES, vs = j % C::V_STAGES;
                if (!wait(bar(C::K_EMPTY + ks), ((uint32_t)(j / C::K_STAGES) & 1u) ^ 1u)) break;
                mbar_expect_tx(bar(C::K_FULL + ks), KV_TILE);
                load_tile(&p.map_k, k_tile + ks * KV_TILE, bar(C::K_FULL + ks), g * D, start + j * KEYS, D, KV_PART);
                if (!wait(bar(C::V_EMPTY + vs), ((uint32_t)(j / C::V_STAGES) & 1u) ^ 1u)) break;
                mbar_expect_tx(bar(C::V_FULL + vs), KV_TILE);
                load_tile(&p.map_v, v_tile + vs * KV_TILE, bar(C::V_FULL + vs), g * D, start + j * KEYS, D, KV_PART);
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t idesc_s = make_idesc<false, false, 128>(KEYS), idesc_dq = make_idesc<false, true, 128>(D);
            const uint64_t q_desc = make_desc(q_tile, 16, 1024), do_desc = make_desc(do_tile, 16, 1024), k_desc = make_desc(k_tile, 16, 1024);
            const uint64_t v_desc = make_desc(v_tile, 16, 1024), k_mn_desc = make_desc(k_tile, KV_PART, 1024);
            auto scores = [&](int j) {      // S = Q K^T of block j into its buffer
                const int st = j % C::K_STAGES;
                if (!wait(bar(C::K_FULL + st), (uint32_t)(j / C::K_STAGES) & 1u)) return false;
                tc_fence_after();
                const uint64_t k_of = k_desc + (uint64_t)(st * (KV_TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma_bf16(tmem + (uint32_t)(j % C::BUFFERS) * KEYS, q_desc + (k_major<PART>(kk) >> 4), k_of + (k_major<KV_PART>(kk) >> 4), idesc_s, kk ? 1u : 0u);
                umma_commit(bar(C::S_FULL + (j & 1)));
                return true;
            };
            auto d_probabilities = [&](int j) {    // dP = dO V^T of block j
                const int st = j % C::V_STAGES;
                if (!wait(bar(C::V_FULL + st), (uint32_t)(j / C::V_STAGES) & 1u)) return false;
                tc_fence_after();
                const uint64_t v_of = v_desc + (uint64_t)(st * (KV_TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) umma_bf16(tmem_dp, do_desc + (k_major<PART>(kk) >> 4), v_of + (k_major<KV_PART>(kk) >> 4), idesc_s, kk ? 1u : 0u);
                umma_commit(bar(C::DP_FULL));
                umma_commit(bar(C::V_EMPTY + st));
                return true;
            };
            auto used = [&](int j) { return wait(bar(C::K_EMPTY + j % C::K_STAGES), (uint32_t)(j / C::K_STAGES) & 1u); };     // the dS of block j has been read
            bool ok = wait(bar(C::Q_FULL), 0) && scores(0) && d_probabilities(0);
            for (int j = 0; ok && j < n; ++j) {
                if (C::BUFFERS == 2) {
                    if (j > 0) ok = used(j - 1);
                    if (ok && j + 1 < n) ok = scores(j + 1);
                } else if (j + 1 < n) {
                    ok = wait(bar(C::S_TAKEN), (uint32_t)j & 1u) && scores(j + 1);
                }
                if (ok) ok = wait(bar(C::DS_FULL), (uint32_t)j & 1u);
                if (!ok) break;
                tc_fence_after();
                if (C::BUFFERS == 2 && j + 1 < n) ok = d_probabilities(j + 1);       // the rows have read this block's dP
                if (!ok) break;
                const int st = j % C::K_STAGES;
                // dQ += dS K: dS from tensor memory, the K tile read as the MN-major operand (rows = key positions)
                const uint64_t k_of = k_mn_desc + (uint64_t)(st * (KV_TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < KEYS / 16; ++kk)
                    umma_bf16_ts(tmem_dq, (C::BUFFERS == 2 ? tmem + (uint32_t)(j % C::BUFFERS) * KEYS : tmem_dp) + p_column<KEYS>(kk), k_of + (uint64_t)(kk * (2048 >> 4)), idesc_dq,
                                 (j | kk) ? 1u : 0u);
                umma_commit(bar(C::K_EMPTY + st));
                if (j == n - 1) umma_commit(bar(C::DQ_DONE));
                if (C::BUFFERS == 1 && j + 1 < n) ok = used(j) && d_probabilities(j + 1);
            }
            if (ok) wait(bar(C::DQ_DONE), 0);         // the last commit has arrived
        }
        __syncwarp();
    } else {
        constexpr int COLS = KEYS;                // columns of a block per thread
        const int quad = warp & 3, row = quad * 32 + lane, tq = i * BLOCK + row;
        const bool live = tq < length;
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const long long at = (start + (long long)(live ? tq : 0)) * p.heads + h;
        // delta = sum_j grad_out * out of this row (kept for the dk, dv kernel): a row to D / 8 lanes, in 16-byte pieces
        constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;
        float delta = 0.f, lse2 = 0.f;
        if (live) lse2 = p.lse[at] * LOG2E;
        {
            uint4 a[8], o[8];
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += 8 * AT_ONCE) {
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int t = i * BLOCK + quad * 32 + r0 + r * AT_ONCE + lane / LANES;
                    const long long piece = ((start + (long long)(t < length ? t : 0)) * p.heads + h) * LANES + lane % LANES;
                    a[r] = reinterpret_cast<const uint4*>(p.grad_out)[piece];
                    o[r] = reinterpret_cast<const uint4*>(p.out_in)[piece];
                }
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    float sum = dot8(a[r], o[r], 0.f);
#pragma unroll
                    for (int w = 1; w < LANES; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
                    // every lane of a row has its sum: lane r0 + r AT_ONCE + x takes that of row group x
                    const float mine = __shfl_sync(0xffffffffu, sum, lane % AT_ONCE * LANES);
                    if (lane / AT_ONCE == r0 / AT_ONCE + r) delta = mine;
                }
            }
            if (live) p.delta[at] = delta;
            else delta = 0.f;
        }
        const float scale2 = p.scale * LOG2E;
        const uint64_t scale_pair = pair2(scale2, scale2), lse_pair = pair2(-lse2, -lse2);
        uint64_t delta_pair = pair2(-delta, -delta);
        // The output that delta is formed from was rounded, which counts for queries that see few keys: their dP and delta nearly cancel (a first position's
        // do entirely).  Queries that see keys of the first block alone take delta from the products themselves, sum_s P dP.
        const bool few_keys = i == 0 && quad < KEYS / 32;
        bool ok = true;
        for (int j = 0; ok && j < n; ++j) {
            const uint32_t tmem_s = tmem + (uint32_t)(j % C::BUFFERS) * KEYS + lane_base;
            const int first = j * KEYS - i * BLOCK;                     // first key position of the block, from the CTA's first query
            const bool masked = first + COLS - 1 > quad * 32;            // some row of this warp may not see some of these columns
            uint32_t s[COLS], dp[COLS], packed[COLS / 2];
            ok = wait.all(bar(C::S_FULL + (j & 1)), (uint32_t)(j >> 1) & 1u);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < COLS; c += 32) tmem_ld32(tmem_s + c, s + c);
            tmem_ld_wait();
            if (C::BUFFERS == 1) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(C::S_TAKEN));
            }
#pragma unroll
            for (int c = 0; c < COLS; c += 2) {
                const uint64_t x = fma2(pair2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale_pair, lse_pair);
                float x0, x1;
                if ((c >> 1) % ON_FMA == ON_FMA - 1) {
                    exp2_two(x, x0, x1);
                } else {
                    unpair2(x, x0, x1);
                    x0 = exp2_fast(x0);
                    x1 = exp2_fast(x1);
                }
                s[c] = __float_as_uint(x0);
                s[c + 1] = __float_as_uint(x1);
            }
            ok = wait.all(bar(C::DP_FULL), (uint32_t)j & 1u);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < COLS; c += 32) tmem_ld32(tmem_dp + lane_base + c, dp + c);
            tmem_ld_wait();
            if (few_keys && j == 0) {
                float sum[4] = {};
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    if (c <= row) sum[c & 3] = fmaf(__uint_as_float(s[c]), __uint_as_float(dp[c]), sum[c & 3]);
                delta = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                delta_pair = pair2(-delta, -delta);
                if (live) p.delta[at] = delta;
            }
            // dS without the scale of the scores, which the last step applies to dQ
#pragma unroll
            for (int c = 0; c < COLS; c += 2) {
                float d0, d1;
                unpair2(mul2(pair2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])),
                             add2(pair2(__uint_as_float(dp[c]), __uint_as_float(dp[c + 1])), delta_pair)), d0, d1);
                s[c] = __float_as_uint(d0);
                s[c + 1] = __float_as_uint(d1);
            }
            if (masked) {      // a loop of its own: the mask costs the blocks on the diagonal alone
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    if (first + c > row) s[c] = 0u;
            }
#pragma unroll
            for (int c = 0; c < COLS; c += 2) packed[c >> 1] = pack2(__uint_as_float(s[c]), __uint_as_float(s[c + 1]));
            tmem_st32(C::BUFFERS == 2 ? tmem_s : tmem_dp + lane_base, packed);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::DS_FULL));
        }
        if (ok) ok = wait.all(bar(C::DQ_DONE), 0);
        if (ok) {
            tc_fence_after();
            float odd = 0.f;
            uint4* dst = reinterpret_cast<uint4*>(p.out + at * D);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                tmem_ld32(tmem_dq + lane_base + c * 32, r);
                tmem_ld_wait();
                odd += oddness(r);
                if (live) store_row32(dst + c * 4, r, p.scale);
            }
            if (live && odd != 0.f && lse2 == lse2 && delta == delta) dq_again<D>(p, start, tq, h, g, lse2, delta);
        }
    }
    linger_after_abort(&s_abort);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        release(tmem, 256);
    }
}

// ------------------------------------------------------------------------------------------------
// backward, part 2: dk and dv, a CTA to 128 keys of a key/value head and, where those are too few to fill the machine, a cluster of `p.split`
// CTAs that share its (query head, query block) list and add their dk, dv through distributed shared memory in a fixed order
// ------------------------------------------------------------------------------------------------
constexpr int DKV_ROW_BYTES = 2 * BLOCK * 4;           // -lse * log2 e and -delta of a query block
template <int D> struct DKV {
    static constexpr int PART = BLOCK * 128, TILE = D / 64 * PART;
    static constexpr int STAGES = D == 64 ? 3 : 2;
    static constexpr int BUFFERS = D == 64 ? 2 : 1;                             // of S^T
    static constexpr int TILES = (2 + 2 * STAGES) * TILE, ROWS_AT = TILES;
    static constexpr int SUM_PITCH = 2 * D * 4 + 16;                            // a row of dv and dk sums; 16 more bytes spread the rows over the banks
    static_assert(BLOCK * SUM_PITCH <= TILES, "the sums fit where the tiles were");
    enum { KV_FULL = 0, Q_FULL = 1, Q_EMPTY = Q_FULL + STAGES, DO_FULL = Q_EMPTY + STAGES, DO_EMPTY = DO_FULL + STAGES, S_FULL = DO_EMPTY + STAGES, DP_FULL = S_FULL + 2,
           P_FULL, DS_FULL = P_FULL + 2, ACC_DONE, BARS };
    static constexpr int BARS_AT = ROWS_AT + STAGES * DKV_ROW_BYTES;
    static constexpr int SMEM = BARS_AT + 8 * BARS + 24;
};

template <int D>
__global__ void __launch_bounds__(DKV_THREADS, 1)
packed_dkv_kernel(const __grid_constant__ PackedParams p) {
    using C = DKV<D>;
    constexpr int TILE = C::TILE, PART = C::PART, STAGES = C::STAGES, CHUNKS = 2 * D / 32;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem_raw);
    const uint32_t k_tile = base, v_tile = base + TILE, q_tile = v_tile + TILE, do_tile = q_tile + STAGES * TILE;
    const uint32_t rows_at = base + C::ROWS_AT, bars = base + C::BARS_AT;
    // the first `shared` lists, the longest, are cut among a cluster's CTAs; behind them every CTA has a list of its own
    const int cluster = (int)blockIdx.x / p.split, place = (int)blockIdx.x % p.split;
    const bool cut = cluster < p.shared;
    const int job = cut ? cluster : p.shared + (cluster - p.shared) * p.split + place, share = cut ? place : 0, split = cut ? p.split : 1;
    if (job >= p.jobs) {      // the last cluster has more CTAs than there are lists
        chain_wait();
        return;
    }
    // S_FULL and P_FULL are two barriers each, by the parity of the iteration (attention.cu says why)
    auto bar = [&](int which) { return bars + 8u * which; };
    uint32_t& s_tmem_base = *reinterpret_cast<uint32_t*>(smem_raw + C::BARS_AT + 8 * C::BARS);
    volatile int& s_abort = *reinterpret_cast<volatile int*>(smem_raw + C::BARS_AT + 8 * C::BARS + 4);
    int* s_item = reinterpret_cast<int*>(smem_raw + C::BARS_AT + 8 * C::BARS + 8);
    if (base & 1023u) {
        chain_wait();
        if (threadIdx.x == 0) atomicExch(p.status, STATUS_ATTENTION_WAIT + 1);
        return;
    }
    if (threadIdx.x == 0) {
        s_abort = 0;
        // a stage is full when its bytes have landed and the lanes of the loading warp have written its row values
        for (int w = 0; w < C::BARS; ++w) {
            const bool rows = w >= C::P_FULL && w <= C::DS_FULL, full = w >= C::Q_FULL && w < C::Q_EMPTY;
            mbar_init(bar(w), rows ? 4 * DKV_PARTS : full ? 2 : 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&p.map_q); prefetch_map(&p.map_k); prefetch_map(&p.map_v); prefetch_map(&p.map_do);
    }
    if (warp == 1) allocate(&s_tmem_base, 512);
    if (warp == 2) fetch_item(p, job / p.kv_heads, s_item);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    chain_wait();
    chain_next();      // the tensor memory is this block's
    const int start = uniform(s_item[0]), length = uniform(s_item[1]), blocks = (length + BLOCK - 1) / BLOCK;
    const int j = blocks - 1 - uniform(s_item[2]);                         // the list's block with the most key blocks is the one with the most query blocks
    const int g = job % p.kv_heads, group = p.heads / p.kv_heads;
    const int per_head = blocks - j;                           // query blocks j .. blocks - 1
    const int all = group * per_head;                          // iterations: head of the group (outer), query block (inner)
    const int begin = (int)((long long)all * share / split), n = (int)((long long)all * (share + 1) / split) - begin;     // this CTA's
    const int first_head = begin / per_head, first_i = j + begin % per_head;
    const uint32_t tmem = s_tmem_base;
    // everything with key positions as rows (lanes) and query positions as columns: S^T of iteration it in columns 128 (it % BUFFERS) ..
    const uint32_t tmem_dp = tmem + C::BUFFERS * 128, tmem_dv = tmem_dp + 128, tmem_dk = tmem_dv + D;
    const QuickWait wait{{&s_abort, p.status}};

    if (n == 0) {
        // nothing to do before the sum
    } else if (warp == 0) {
        if (lane == 0) {
            mbar_expect_tx(bar(C::KV_FULL), 2 * TILE);
            load_tile(&p.map_k, k_tile, bar(C::KV_FULL), g * D, start + j * BLOCK, D, PART);
            load_tile(&p.map_v, v_tile, bar(C::KV_FULL), g * D, start + j * BLOCK, D, PART);
        }
        int st = 0, head = first_head, i = first_i;
        uint32_t parity = 1;
        float lse2[BLOCK / 32], delta[BLOCK / 32];
        auto fetch_rows = [&] {        // the row values of a query block; past the sequence's end a probability of zero
#pragma unroll
            for (int r = 0; r < BLOCK / 32; ++r) {
                const int tq = i * BLOCK + r * 32 + lane;
                const long long at = (start + (long long)tq) * p.heads + g * group + head;
                lse2[r] = tq < length ? -p.lse[at] * LOG2E : -INFINITY;
                delta[r] = tq < length ? -p.delta[at] : 0.f;
            }
        };
        bool ok = true;
        for (int it = 0; ok && it < n; ++it) {
            const int h = g * group + head;
            // dO is done with before Q is (dV before dK), and comes before it
            ok = wait.all(bar(C::DO_EMPTY + st), parity);
            if (!ok) break;
            if (lane == 0) {
                mbar_expect_tx(bar(C::DO_FULL + st), TILE);
                load_tile(&p.map_do, do_tile + st * TILE, bar(C::DO_FULL + st), h * D, start + i * BLOCK, D, PART);
            }
            ok = wait.all(bar(C::Q_EMPTY + st), parity);
            if (!ok) break;
            if (lane == 0) {
                mbar_expect_tx(bar(C::Q_FULL + st), TILE);
                load_tile(&p.map_q, q_tile + st * TILE, bar(C::Q_FULL + st), h * D, start + i * BLOCK, D, PART);
            }
            if (it == 0) fetch_rows();
            float* rows = reinterpret_cast<float*>(smem_raw + C::ROWS_AT + st * DKV_ROW_BYTES);
#pragma unroll
            for (int r = 0; r < BLOCK / 32; ++r) {
                rows[r * 32 + lane] = lse2[r];
                rows[BLOCK + r * 32 + lane] = delta[r];
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::Q_FULL + st));
            if (++st == STAGES) { st = 0; parity ^= 1u; }
            if (++i == blocks) { i = j; ++head; }
            if (it + 1 < n) fetch_rows();        // the next ones travel while their stage is still in use
        }
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t idesc_s = make_idesc<false, false, 128>(128), idesc_t = make_idesc<false, true, 128>(D);
            const uint64_t k_desc = make_desc(k_tile, 16, 1024), v_desc = make_desc(v_tile, 16, 1024), q_desc = make_desc(q_tile, 16, 1024);
            const uint64_t do_desc = make_desc(do_tile, 16, 1024), q_mn_desc = make_desc(q_tile, PART, 1024), do_mn_desc = make_desc(do_tile, PART, 1024);
            auto scores = [&](int it) {      // S^T = K Q^T
                const int st = it % STAGES;
                if (!wait(bar(C::Q_FULL + st), (uint32_t)(it / STAGES) & 1u)) return false;
                tc_fence_after();
                const uint64_t q_of = q_desc + (uint64_t)(st * (TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma_bf16(tmem + (uint32_t)(it % C::BUFFERS) * 128, k_desc + (k_major<PART>(kk) >> 4), q_of + (k_major<PART>(kk) >> 4), idesc_s, kk ? 1u : 0u);
                umma_commit(bar(C::S_FULL + (it & 1)));
                return true;
            };
            auto d_probabilities = [&](int it) {    // dP^T = V dO^T
                const int st = it % STAGES;
                if (!wait(bar(C::DO_FULL + st), (uint32_t)(it / STAGES) & 1u)) return false;
                tc_fence_after();
                const uint64_t do_of = do_desc + (uint64_t)(st * (TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) umma_bf16(tmem_dp, v_desc + (k_major<PART>(kk) >> 4), do_of + (k_major<PART>(kk) >> 4), idesc_s, kk ? 1u : 0u);
                umma_commit(bar(C::DP_FULL));
                return true;
            };
            auto used = [&](int it) { return wait(bar(C::Q_EMPTY + it % STAGES), (uint32_t)(it / STAGES) & 1u); };     // all products of iteration it are done
            bool ok = wait(bar(C::KV_FULL), 0) && scores(0) && d_probabilities(0);
            for (int it = 0; ok && it < n; ++it) {
                const int st = it % STAGES;
                const uint32_t buffer = tmem + (uint32_t)(it % C::BUFFERS) * 128;
                if (C::BUFFERS == 2) {
                    if (it > 0) ok = used(it - 1);
                    if (ok && it + 1 < n) ok = scores(it + 1);
                }
                if (ok) ok = wait(bar(C::P_FULL + (it & 1)), (uint32_t)(it >> 1) & 1u);
                if (!ok) break;
                tc_fence_after();
                // dV += P^T dO and dK += dS^T Q: P^T and dS^T from tensor memory, dO and Q as they lie in memory (rows = query
                // positions = the contraction) are MN-major operands
                const uint64_t do_of = do_mn_desc + (uint64_t)(st * (TILE >> 4)), q_of = q_mn_desc + (uint64_t)(st * (TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < BLOCK / 16; ++kk)
                    umma_bf16_ts(tmem_dv, buffer + p_column<BLOCK / DKV_PARTS>(kk), do_of + (uint64_t)(kk * (2048 >> 4)), idesc_t, (it | kk) ? 1u : 0u);
                umma_commit(bar(C::DO_EMPTY + st));
                if (C::BUFFERS == 1 && it + 1 < n) ok = wait(bar(C::DO_EMPTY + st), (uint32_t)(it / STAGES) & 1u) && scores(it + 1);      // P has been read
                if (ok) ok = wait(bar(C::DS_FULL), (uint32_t)it & 1u);
                if (!ok) break;
                tc_fence_after();
                if (C::BUFFERS == 2 && it + 1 < n) ok = d_probabilities(it + 1);     // the rows have read this iteration's dP, and put dS elsewhere
                if (!ok) break;
                const uint32_t ds = C::BUFFERS == 2 ? buffer + BLOCK / DKV_PARTS / 2 : tmem_dp;
#pragma unroll
                for (int kk = 0; kk < BLOCK / 16; ++kk)
                    umma_bf16_ts(tmem_dk, ds + p_column<BLOCK / DKV_PARTS>(kk), q_of + (uint64_t)(kk * (2048 >> 4)), idesc_t, (it | kk) ? 1u : 0u);
                umma_commit(bar(C::Q_EMPTY + st));
                if (it == n - 1) umma_commit(bar(C::ACC_DONE));
                if (C::BUFFERS == 1 && it + 1 < n) ok = used(it) && d_probabilities(it + 1);
            }
            if (ok) wait(bar(C::ACC_DONE), 0);        // the last commit has arrived
        }
        __syncwarp();
    } else {
        constexpr int COLS = BLOCK / DKV_PARTS;    // columns (query positions) of a block per thread
        const int quad = warp & 3, row = quad * 32 + lane, part = (warp - 2) >> 2;
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        const float scale2 = p.scale * LOG2E;
        const uint64_t scale_pair = pair2(scale2, scale2);
        int st = 0, i = first_i;
        bool ok = true;
        for (int it = 0; ok && it < n; ++it) {
            const uint32_t tmem_s = tmem + (uint32_t)(it % C::BUFFERS) * 128 + lane_base + part * COLS;
            const uint32_t row_values = rows_at + st * DKV_ROW_BYTES + part * COLS * 4;
            const bool masked = i == j && part * COLS < quad * 32 + 31;  // some row of this warp is not seen by some of these columns
            const int live = length - i * BLOCK - part * COLS;           // columns from here on are past the end of the sequence
            uint32_t s[COLS], dp[COLS];
            auto put_back = [&](uint32_t to) {         // s, rounded to bf16, 32 columns at a time (the registers of all at once spill)
#pragma unroll
                for (int c = 0; c < COLS; c += 32) {
                    uint32_t packed[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) packed[e >> 1] = pack2(__uint_as_float(s[c + e]), __uint_as_float(s[c + e + 1]));
                    tmem_st16(to + c / 2, packed);
                }
            };
            auto clear_unseen = [&] {
                if (masked) {
#pragma unroll
                    for (int c = 0; c < COLS; ++c)
                        if (part * COLS + c < row) s[c] = 0u;
                }
                if (live < COLS) {
#pragma unroll
                    for (int c = 0; c < COLS; ++c)
                        if (c >= live) s[c] = 0u;
                }
            };
            ok = wait.all(bar(C::Q_FULL + st), (uint32_t)(it / STAGES) & 1u);      // publishes the row values of this stage
            if (ok) ok = wait.all(bar(C::S_FULL + (it & 1)), (uint32_t)(it >> 1) & 1u);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < COLS; c += 32) tmem_ld32(tmem_s + c, s + c);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < COLS; c += 4) {
                float l[4], x[4];
                load_shared4(row_values + c * 4, l);
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    unpair2(fma2(pair2(__uint_as_float(s[c + e]), __uint_as_float(s[c + e + 1])), scale_pair, pair2(l[e], l[e + 1])), x[e], x[e + 1]);
                    s[c + e] = __float_as_uint(exp2_fast(x[e]));
                    s[c + e + 1] = __float_as_uint(exp2_fast(x[e + 1]));
                }
            }
            clear_unseen();
            put_back(tmem_s);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::P_FULL + (it & 1)));
            ok = wait.all(bar(C::DP_FULL), (uint32_t)it & 1u);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < COLS; c += 32) tmem_ld32(tmem_dp + lane_base + part * COLS + c, dp + c);
            tmem_ld_wait();
            // dS without the scale of the scores, which the last step applies to dK
#pragma unroll
            for (int c = 0; c < COLS; c += 4) {
                float d[4];
                load_shared4(row_values + BLOCK * 4 + c * 4, d);
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    float d0, d1;
                    unpair2(mul2(pair2(__uint_as_float(s[c + e]), __uint_as_float(s[c + e + 1])),
                                 add2(pair2(__uint_as_float(dp[c + e]), __uint_as_float(dp[c + e + 1])), pair2(d[e], d[e + 1]))), d0, d1);
                    s[c + e] = __float_as_uint(d0);
                    s[c + e + 1] = __float_as_uint(d1);
                }
            }
            clear_unseen();         // 0 times the gradient's product with a value that is no number
            put_back(C::BUFFERS == 2 ? tmem_s + COLS / 2 : tmem_dp + lane_base + part * COLS);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::DS_FULL));
            if (++st == STAGES) st = 0;
            if (++i == blocks) i = j;
        }
        if (ok) ok = wait.all(bar(C::ACC_DONE), 0);
        if (ok) {
            tc_fence_after();
            const int tk = j * BLOCK + row;                     // this thread's key position
            const long long at = (start + (long long)(tk < length ? tk : 0)) * p.kv_heads + g;
#pragma unroll 1
            for (int c = part; c < CHUNKS; c += DKV_PARTS) {    // 32-column chunks, dv's first, dk's behind
                uint32_t r[32];
                tmem_ld32(tmem_dv + lane_base + c * 32, r);
                tmem_ld_wait();
                const bool is_dk = c >= CHUNKS / 2;
                if (tk < length && oddness(r) != 0.f) {
                    uint32_t again[32];
                    dkv_again<D>(p, start, length, tk, g, j, first_head, first_i, n, c, again);
#pragma unroll
                    for (int e = 0; e < 32; ++e) r[e] = again[e];
                }
                __syncwarp();
                if (split > 1) {      // the tiles of this CTA are spent: its sums take their place
                    float4* sums = reinterpret_cast<float4*>(smem_raw + row * C::SUM_PITCH + c * 128);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        sums[e] = make_float4(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1]), __uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3]));
                } else if (tk < length) {
                    store_row32(reinterpret_cast<uint4*>((is_dk ? p.out : p.out2) + at * D) + c % (CHUNKS / 2) * 4, r, is_dk ? p.scale : 1.f);
                }
            }
        }
    }
    linger_after_abort(&s_abort);
    tc_fence_before();
    if (split > 1) {
        cluster_sync();
        // every CTA adds the sums of all for its share of the 128 rows, in pieces of 8 columns (dv's first, dk's behind)
        constexpr int PIECES = 2 * D / 8;
        const int row0 = BLOCK * share / split, rows = BLOCK * (share + 1) / split - row0;
        for (int at = threadIdx.x; at < rows * PIECES; at += DKV_THREADS) {
            const int row = row0 + at / PIECES, piece = at % PIECES, tk = j * BLOCK + row;
            float total[8] = {}, v[8][8];
#pragma unroll
            for (int other = 0; other < 8; ++other) {        // all on their way before the first is added
#pragma unroll
                for (int e = 0; e < 8; ++e) v[other][e] = 0.f;
                if (other >= split || (all < split && all * (other + 1) / split == all * other / split)) continue;        // none, or without iterations
                const uint32_t from = map_to_cta(base + row * C::SUM_PITCH + piece * 32, other);
                load_cluster4(from, v[other]);
                load_cluster4(from + 16, v[other] + 4);
            }
#pragma unroll
            for (int other = 0; other < 8; ++other)
#pragma unroll
                for (int e = 0; e < 8; ++e) total[e] += v[other][e];
            const bool is_dk = piece >= PIECES / 2;
            const float scale = is_dk ? p.scale : 1.f;
            if (tk < length)
                reinterpret_cast<uint4*>((is_dk ? p.out : p.out2) + ((start + (long long)tk) * p.kv_heads + g) * D)[piece % (PIECES / 2)] =
                    make_uint4(pack2(total[0] * scale, total[1] * scale), pack2(total[2] * scale, total[3] * scale),
                               pack2(total[4] * scale, total[5] * scale), pack2(total[6] * scale, total[7] * scale));
        }
        cluster_sync();        // nobody leaves while its sums are being read
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        release(tmem, 512);
    }
}

// CTAs per key block of the dk, dv kernel.  More of them shorten the longest list (every query block of every head of the group) and cost each CTA its
// start and end once more, the ends with sums through distributed shared memory: in iterations (1.4 us with heads of 64, 2.2 with 128) 4 and 3 for a
// CTA by itself, 9 and 7 for one of a cluster.  Forward and backward in us with 1, 2, 4 and 8: five documents of up to 130 positions, 8 heads of 64 in 2 groups,
// 38, 37, 32 and 30; 17 documents of up to 2048, 16 heads of 64 in 4 groups, 170, 178, 241 and 389; six of up to 1999, 8 heads of 128, 107, 136, 222 and 432.
// The same rule says whether all lists are cut or those alone that are longer than the longest one's share: then the second case takes 157 in clusters of 2, of which 48 lists have
// one each and 244 half of one.  (Measured with a forward some 5 us shorter in the second and third case.)
struct Cut { int split; long long shared; };
Cut packed_split(const qmoe_packed_attention_t* a) {
    const double alone = a->dim == 64 ? 4 : 3, shared = a->dim == 64 ? 9 : 7, slots = sm_count();
    const double longest = (double)(a->heads / a->kv_heads) * a->longest, share = (double)a->pairs * a->heads / slots, jobs = (double)a->blocks * a->kv_heads;
    const int64_t above[4] = {0, a->above_half, a->above_quarter, a->above_eighth};
    Cut best = {1, 0};
    double least = 0;
    for (int i = 0, split = 1; i < 4 && (split == 1 || longest >= split); ++i, split *= 2) {
        for (const long long items : {(long long)a->blocks, (long long)above[i]}) {
            if (split > 1 && items <= 0) continue;
            const double lists = split > 1 ? (double)items * a->kv_heads : 0;
            const double critical = longest / split + (split > 1 ? shared : alone), busy = share + (shared * lists * split + alone * (jobs - lists)) / slots;
            const double cost = critical > busy ? critical : busy;
            if (split == 1 || cost < least) { least = cost; best = {split, (long long)lists}; }
            if (split == 1) break;
        }
    }
    return best;
}

int packed_check(const qmoe_packed_attention_t* a, bool backward) {
    if (!a) return fail_arg("packed attention: argument is null");
    if (a->dim != 64 && a->dim != 128) return fail_arg("packed attention: the head width must be 64 or 128");
    if (a->dtype != QMOE_BF16) return fail_arg("packed attention: dtype must be QMOE_BF16");
    if (a->rows <= 0 || a->blocks <= 0 || a->longest <= 0 || a->pairs <= 0) return fail_arg("packed attention: there must be rows");
    if (a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads) return fail_arg("packed attention: heads must be a positive multiple of kv_heads");
    if (a->heads > (1 << 16) || a->rows > 0x7fffff00ll - BLOCK || a->blocks > a->rows || a->longest > a->blocks || a->blocks * a->heads > 0x0fffffffll)
        return fail_arg("packed attention: too many rows, blocks or heads");
    for (const int64_t above : {a->above_half, a->above_quarter, a->above_eighth})
        if (above < 0 || above > a->blocks) return fail_arg("packed attention: more long entries than entries");
    if (!(a->scale > 0) || a->scale > 1e30f) return fail_arg("packed attention: the scale must be a positive number");
    if (!a->q || !a->k || !a->v || !a->out || !a->lse || !a->table) return fail_arg("packed attention: null buffer address");
    if (backward && (!a->grad_out || !a->delta || !a->dq || !a->dk || !a->dv)) return fail_arg("packed attention: null buffer address");
    if ((a->q | a->k | a->v | a->out | a->grad_out | a->dq | a->dk | a->dv | a->table) & 15u || (a->lse | a->delta) & 3u)
        return fail_arg("packed attention: buffers must be 16-byte aligned");
    const int64_t wide = (int64_t)a->heads * a->dim, narrow = (int64_t)a->kv_heads * a->dim, most = 1ll << 31;
    if ((a->q_pitch | a->k_pitch | a->v_pitch) % 8 || a->q_pitch < wide || a->k_pitch < narrow || a->v_pitch < narrow || a->q_pitch > most || a->k_pitch > most ||
        a->v_pitch > most)
        return fail_arg("packed attention: a row pitch must be a multiple of 16 bytes and not below the row's width");
    // a CTA's outputs are other CTAs' operands nowhere
    struct Span { uint64_t at, bytes; };
    const uint64_t rows = (uint64_t)a->rows;
    auto pitched = [&](uint64_t at, int64_t pitch, int64_t width) { return Span{at, ((rows - 1) * (uint64_t)pitch + (uint64_t)width) * 2}; };
    const Span in[] = {pitched(a->q, a->q_pitch, wide), pitched(a->k, a->k_pitch, narrow), pitched(a->v, a->v_pitch, narrow), pitched(backward ? a->out : 0, wide, wide),
                       pitched(backward ? a->grad_out : 0, wide, wide), {backward ? a->lse : 0, rows * a->heads * 4}, {a->table, (uint64_t)a->blocks * 16}};
    const Span out[] = {pitched(backward ? a->dq : a->out, wide, wide), {backward ? a->delta : a->lse, rows * a->heads * 4}, pitched(backward ? a->dk : 0, narrow, narrow),
                        pitched(backward ? a->dv : 0, narrow, narrow)};
    auto overlap = [](const Span& x, const Span& y) { return x.at && y.at && x.at < y.at + y.bytes && y.at < x.at + x.bytes; };
    for (int i = 0; i < 4; ++i) {
        for (const Span& read : in)
            if (overlap(out[i], read)) return fail_arg("packed attention: an output overlaps an operand");
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) return fail_arg("packed attention: two outputs overlap");
    }
    return 0;
}

PackedParams packed_params(const qmoe_packed_attention_t* a) {
    PackedParams p = {};
    p.items = (const int4*)a->table;
    p.q = (const __nv_bfloat16*)a->q; p.k = (const __nv_bfloat16*)a->k; p.v = (const __nv_bfloat16*)a->v;
    p.lse = (float*)a->lse; p.delta = (float*)a->delta; p.status = device_status_address();
    p.q_pitch = a->q_pitch; p.k_pitch = a->k_pitch; p.v_pitch = a->v_pitch;
    p.scale = a->scale; p.heads = a->heads; p.kv_heads = a->kv_heads; p.split = 1;
    return p;
}

template <int D> int packed_forward(const qmoe_packed_attention_t* a, cudaStream_t stream) {
    PackedParams p = packed_params(a);
    const uint64_t wide = (uint64_t)a->heads * D, narrow = (uint64_t)a->kv_heads * D, rows = (uint64_t)a->rows;
    if (int rc = make_map_2d(&p.map_q, a->q, wide, rows, BLOCK, a->q_pitch)) return rc;
    if (int rc = make_map_2d(&p.map_k, a->k, narrow, rows, KEYS, a->k_pitch)) return rc;
    if (int rc = make_map_2d(&p.map_v, a->v, narrow, rows, KEYS, a->v_pitch)) return rc;
    p.out = (__nv_bfloat16*)a->out;
    QMOE_CUDA(allow_shared<packed_forward_kernel<D>>(Forward<D>::SMEM));
    chained(packed_forward_kernel<D>, (unsigned)(a->blocks * a->heads), THREADS, Forward<D>::SMEM, stream, p);
    count_tensor_core_launch();
    QMOE_LAUNCH_CHECK("packed_forward_kernel");
    return 0;
}

template <int D> int packed_backward(const qmoe_packed_attention_t* a, cudaStream_t stream) {
    PackedParams p = packed_params(a);
    const uint64_t wide = (uint64_t)a->heads * D, narrow = (uint64_t)a->kv_heads * D, rows = (uint64_t)a->rows;
    if (int rc = make_map_2d(&p.map_q, a->q, wide, rows, BLOCK, a->q_pitch)) return rc;
    if (int rc = make_map_2d(&p.map_do, a->grad_out, wide, rows, BLOCK)) return rc;
    if (int rc = make_map_2d(&p.map_k, a->k, narrow, rows, KEYS, a->k_pitch)) return rc;
    if (int rc = make_map_2d(&p.map_v, a->v, narrow, rows, KEYS, a->v_pitch)) return rc;
    p.out_in = (const __nv_bfloat16*)a->out; p.grad_out = (const __nv_bfloat16*)a->grad_out;
    p.out = (__nv_bfloat16*)a->dq;
    QMOE_CUDA(allow_shared<packed_dq_kernel<D>>(DQ<D>::SMEM));
    QMOE_CUDA(allow_shared<packed_dkv_kernel<D>>(DKV<D>::SMEM));
    chained(packed_dq_kernel<D>, (unsigned)(a->blocks * a->heads), THREADS, DQ<D>::SMEM, stream, p);
    count_tensor_core_launch();
    QMOE_LAUNCH_CHECK("packed_dq_kernel");
    if (int rc = make_map_2d(&p.map_k, a->k, narrow, rows, BLOCK, a->k_pitch)) return rc;
    if (int rc = make_map_2d(&p.map_v, a->v, narrow, rows, BLOCK, a->v_pitch)) return rc;
    p.out = (__nv_bfloat16*)a->dk; p.out2 = (__nv_bfloat16*)a->dv;
    const Cut cut = packed_split(a);
    const long long jobs = a->blocks * a->kv_heads;
    p.split = cut.split; p.shared = (int)cut.shared; p.jobs = (int)jobs;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attributes[2] = {chain_attribute()};
    config.gridDim = dim3((unsigned)((cut.shared + (jobs - cut.shared + cut.split - 1) / cut.split) * cut.split));
    config.blockDim = dim3(DKV_THREADS);
    config.dynamicSmemBytes = DKV<D>::SMEM;
    config.stream = stream;
    config.attrs = attributes;
    config.numAttrs = p.split > 1 ? 2 : 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = (unsigned)p.split;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    QMOE_CUDA(cudaLaunchKernelEx(&config, packed_dkv_kernel<D>, p));
    count_tensor_core_launch();
    QMOE_LAUNCH_CHECK("packed_dkv_kernel");
    return 0;
}

}  // namespace
}  // namespace qmoe

using namespace qmoe;

extern "C" int qmoe_packed_attention_forward(const qmoe_packed_attention_t* a, uint64_t stream_) {
    if (int rc = packed_check(a, false)) return rc;
    cudaStream_t stream = (cudaStream_t)stream_;
    TimedScope timed(KC_ATTENTION, stream);
    return a->dim == 64 ? packed_forward<64>(a, stream) : packed_forward<128>(a, stream);
}

extern "C" int qmoe_packed_attention_backward(const qmoe_packed_attention_t* a, uint64_t stream_) {
    if (int rc = packed_check(a, true)) return rc;
    cudaStream_t stream = (cudaStream_t)stream_;
    TimedScope timed(KC_ATTENTION, stream);
    return a->dim == 64 ? packed_backward<64>(a, stream) : packed_backward<128>(a, stream);
}
