// AdamW over many tensors in one launch with both moments in 8 bits.  Per element, in fp32 (each product and sum rounded by itself, so
// that what is rounded to 8 bits does not depend on how a compiler contracts):
//     m = b1 m + (1 - b1) g,   v = b2 r r + (1 - b2) g g,   p = p (1 - lr decay) - lr / c1 * m / (sqrt(v) / sqrt(c2) + eps),
// (where v would leave the range of fp32, its root is formed from scaled operands: gradients from 1e-19 on up to the largest number have a root)
// with the new m and r = sqrt(v) then held as 8-bit codes times a scale of their block of 256 elements:
//   * m as an e4m3 number, the block's largest |m| at 448: half a step is 2^-4 of a value, down to 2^-15 of the largest;
//   * the root of v, which is what divides, without a sign in 4 exponent and 4 mantissa bits: code c below 16 is c, from there on
//     (16 + c % 16) 2^(c / 16 - 1), the block's largest at 491520 = code 254; half a step is 2^-5, down to 2^-14 of the largest.  A positive root never
//     becomes 0: it divides, and an m whose code is not 0 would be sent far away.  (A linear code of 8 bits leaves nothing below 1 / 255 of the largest.)
// Rounding is to nearest, ties to the even code.  The scale is a float of its own for each block, so that a block's decay between large gradients is
// followed although no code changes.  A moment that is no finite number has a code of its own (0x7f, 255) and no part in the scale.
//
// A warp has two blocks of 256, eight elements of each to a lane, with all their loads in flight.  Bytes an element: p 8, g 4, moments 4, scales 1/16, the bf16
// copy 2: 18 against 30 with moments in 32 bits (optim.cu).
// What bounds it: memory, and near it the issue of instructions (59 % of the cycles: codes to numbers and back).  266 million elements in 92 tensors with their bf16
// copies, and both moments written out as numbers behind the step: 1.46 ms for 7.4 GB, 5.1 TB/s.  One block to a warp 1.61, streaming loads and stores 1.49; the last blocks'
// loads without branches took 156 registers and 1.86.  A block in which some element has had no gradient but zeros (an expert without tokens, an unused token's
// row) or squares beyond the range takes the longer form: 134 million elements in 419 us without such blocks, 652 with a zero in every block, 708 with nothing but zeros.
#include "common.cuh"

#include <cuda_fp8.h>
#include <algorithm>
#include <math.h>
#include <memory>
#include <new>
#include <string.h>

namespace qmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;             // elements that share a scale
constexpr int kChunk = 4096;            // elements of a work unit: two blocks to a warp
constexpr float kAverageTop = 448.f, kRootTop = 491520.f;

struct Item {  // = qmoe_byte_item_t
    float* values;
    const float* grad;
    uint8_t* average;
    float* average_scale;
    uint8_t* root;
    float* root_scale;
    __nv_bfloat16* shadow;
    float* average_out;
    float* square_out;
    long long size;
    long long first_chunk;
    float step, root_factor;
    long long* count;                   // steps taken, then step and root_factor of the one being taken
    long long number;
};
static_assert(sizeof(Item) == sizeof(qmoe_byte_item_t), "the table layout is part of the C ABI");

constexpr int kFewItems = 32;           // tables of up to this many items travel as the kernel's parameters
struct FewItems { Item item[kFewItems]; };

__device__ __forceinline__ int find_item(const Item* items, int count, long long chunk) {      // the last with first_chunk <= chunk
    int lo = 0, hi = count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (items[mid].first_chunk <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// four e4m3 codes as numbers
__device__ __forceinline__ void average_values(uint32_t codes, float scale, float* v) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * i)), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        v[2 * i] = __fmul_rn(f.x, scale);
        v[2 * i + 1] = __fmul_rn(f.y, scale);
    }
}
__device__ __forceinline__ uint32_t average_codes(const float* m, float inverse) {
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float a = finite(m[2 * i]) ? __fmul_rn(m[2 * i], inverse) : NAN, b = finite(m[2 * i + 1]) ? __fmul_rn(m[2 * i + 1], inverse) : NAN;
        codes |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) << (16 * i);
    }
    return codes;
}
__device__ __forceinline__ float root_value(uint32_t code, float scale) {
    // from 16 on the code's bits are those of a float: exponent and mantissa side by side
    const float v = code < 16 ? (float)code : __uint_as_float((code + 2080u) << 19);
    return code == 255 ? NAN : __fmul_rn(v, scale);
}
__device__ __forceinline__ uint32_t root_code(float r, float inverse) {
    const float q = __fmul_rn(r, inverse);
    const uint32_t bits = __float_as_uint(q);
    const uint32_t high = ((bits + 0x3ffffu + ((bits >> 19) & 1u)) >> 19) - 2080u;
    const uint32_t low = r > 0.f ? max(1, __float2int_rn(q)) : 0;
    return !finite(r) ? 255u : q < 16.f ? low : high;
}

__device__ __forceinline__ uint32_t warp_top(uint32_t bits) { return __reduce_max_sync(0xffffffffu, bits); }      // of floats from 0 on

struct Rates { float b1, one_b1, b2, one_b2, keep, eps; };

// The root of vn = b2 old old + (1 - b2) grad grad; where the squares leave the numbers' range, from operands scaled by a power of two
__device__ __forceinline__ float root_of(float vn, float old, float grad, const Rates& rates) {
    if (vn >= 7.888609052210118e-31f && vn <= 3.4028234663852886e38f) return __fsqrt_rn(vn);
    const bool large = vn > 1.f;
    const float by = large ? 5.421010862427522e-20f : 18446744073709551616.f;      // 2^-64, 2^64
    const float o = old * by, g = grad * by;
    return __fsqrt_rn(__fadd_rn(__fmul_rn(__fmul_rn(o, o), rates.b2), __fmul_rn(__fmul_rn(g, g), rates.one_b2))) * (large ? 18446744073709551616.f : 5.421010862427522e-20f);
}

// A block's largest values, and what follows from them
struct BlockScales { float m_scale, r_scale, m_inverse, r_inverse; };
__device__ __forceinline__ BlockScales block_scales(uint32_t m_top, uint32_t r_top) {
    const float m_largest = __uint_as_float(m_top);
    float r_largest = __uint_as_float(r_top);
    // (the inverse of a smaller scale would not be a number: an average below 2^-100 is none, a root counts as at least that large)
    const bool held = m_largest > 7.888609052210118e-31f;
    if (r_largest > 0.f) r_largest = fmaxf(r_largest, 7.888609052210118e-31f);
    return {held ? __fmul_rn(m_largest, (float)(1.0 / 448.0)) : 0.f, __fmul_rn(r_largest, (float)(1.0 / 491520.0)),
            held ? __fdiv_rn(kAverageTop, m_largest) : 0.f, r_largest > 0.f ? __fdiv_rn(kRootTop, r_largest) : 0.f};
}

// Eight elements of a block to a lane, any values: p, the codes and the block's scales become the new ones.
__device__ __forceinline__ BlockScales step_any(float (*p)[4], const float (*g)[4], uint32_t* am, uint32_t* rm, float a_scale, float r_scale, float step,
                                                float root_factor, const Rates& rates) {
    float m[8], r[8];
    uint32_t m_top = 0, r_top = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        average_values(am[h], a_scale, m + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float old = root_value((rm[h] >> (8 * e)) & 255u, r_scale), grad = g[h][e];
            const float mn = __fadd_rn(__fmul_rn(m[4 * h + e], rates.b1), __fmul_rn(grad, rates.one_b1));
            const float vn = __fadd_rn(__fmul_rn(__fmul_rn(old, old), rates.b2), __fmul_rn(__fmul_rn(grad, grad), rates.one_b2));
            const float rn = root_of(vn, old, grad, rates);
            m[4 * h + e] = mn;
            r[4 * h + e] = rn;
            if (finite(mn)) m_top = max(m_top, __float_as_uint(mn) & 0x7fffffffu);
            if (finite(rn)) r_top = max(r_top, __float_as_uint(rn));
            p[h][e] = p[h][e] * rates.keep - __fdividef(step * mn, fmaf(rn, root_factor, rates.eps));
        }
    }
    const BlockScales scales = block_scales(warp_top(m_top), warp_top(r_top));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        am[h] = average_codes(m + 4 * h, scales.m_inverse);
        rm[h] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) rm[h] |= root_code(r[4 * h + e], scales.r_inverse) << (8 * e);
    }
    return scales;
}

// The same values for a block whose numbers are all finite and whose squares stay in range, in fewer instructions; false where they do not (nothing has
// changed then).  A root's code, shifted to where a float has its exponent and mantissa, is that root times 2^-130 times its scale, the codes below 16 as
// numbers without a leading one; 2^-130 travels in two exact factors, the second in the scale.  Rounding below 16 is an addition of 2^23.
__device__ __forceinline__ bool step_usual(float (*p)[4], const float (*g)[4], uint32_t* am, uint32_t* rm, float a_scale, float r_scale, float step,
                                           float root_factor, const Rates& rates, BlockScales& scales) {
    float m[8], r[8];
    uint32_t m_top = 0, r_top = 0, odd = 0;
    const float r_scale30 = r_scale * 1073741824.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        average_values(am[h], a_scale, m + 4 * h);
        odd |= (~rm[h] - 0x01010101u) & rm[h] & 0x80808080u;                      // a byte of 255
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t code = (e < 3 ? rm[h] << (19 - 8 * e) : rm[h] >> 5) & (255u << 19);
            const float old = __fmul_rn(__fmul_rn(__uint_as_float(code), 1.2676506002282294e30f), r_scale30);      // 2^100, and 2^30 in the scale
            const float grad = g[h][e];
            const float mn = __fadd_rn(__fmul_rn(m[4 * h + e], rates.b1), __fmul_rn(grad, rates.one_b1));
            const float vn = __fadd_rn(__fmul_rn(__fmul_rn(old, old), rates.b2), __fmul_rn(__fmul_rn(grad, grad), rates.one_b2));
            odd |= __float_as_uint(vn) - 0x0d800000u > 0x7f7fffffu - 0x0d800000u;  // outside 2^-100 .. the largest number
            r[4 * h + e] = vn;
            m[4 * h + e] = mn;
            m_top = max(m_top, __float_as_uint(mn) & 0x7fffffffu);
        }
    }
    m_top = warp_top(m_top);
    if (__any_sync(0xffffffffu, odd != 0) || m_top >= 0x7f800000u) return false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        r[i] = __fsqrt_rn(r[i]);
        r_top = max(r_top, __float_as_uint(r[i]));
        p[i >> 2][i & 3] = p[i >> 2][i & 3] * rates.keep - __fdividef(step * m[i], fmaf(r[i], root_factor, rates.eps));
    }
    scales = block_scales(m_top, warp_top(r_top));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t codes = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            codes |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(m[4 * h + 2 * i], scales.m_inverse), __fmul_rn(m[4 * h + 2 * i + 1], scales.m_inverse)),
                                                        __NV_SATFINITE, __NV_E4M3) << (16 * i);
        am[h] = codes;
        codes = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float q = __fmul_rn(r[4 * h + e], scales.r_inverse);
            const uint32_t bits = __float_as_uint(q);
            const uint32_t high = ((bits + 0x3ffffu + ((bits >> 19) & 1u)) >> 19) - 2080u;
            const uint32_t low = max(__float_as_uint(q + 8388608.f) & 255u, 1u);
            codes |= (q < 16.f ? low : high) << (8 * e);
        }
        rm[h] = codes;
    }
    return true;
}

// One warp: blocks of 256 elements of an item from element `base` on, lane l of elements 4 l .. 4 l + 3 of every 128.
template <bool WHOLE>
__device__ __forceinline__ void step_blocks(const Item& it, long long base, const Rates& rates) {
    constexpr int BLOCKS = 2, PARTS = 2 * BLOCKS;
    const int lane = threadIdx.x & 31;
    float p[PARTS][4], g[PARTS][4];
    uint32_t am[PARTS], rm[PARTS];
    float a_scale[BLOCKS], r_scale[BLOCKS];
    // numerator and denominator (rates.eps too) carry a factor of 1/16: the fast quotient is 0 for a denominator beyond 2^126
    const float step = it.step * 0.0625f, root_factor = it.root_factor * 0.0625f;
    auto at = [&](int part) { return base + part * 128 + lane * 4; };
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
        const long long i = at(j);
        if (WHOLE) {
            *reinterpret_cast<float4*>(p[j]) = *reinterpret_cast<const float4*>(it.values + i);
            *reinterpret_cast<float4*>(g[j]) = *reinterpret_cast<const float4*>(it.grad + i);
            am[j] = *reinterpret_cast<const uint32_t*>(it.average + i);
            rm[j] = *reinterpret_cast<const uint32_t*>(it.root + i);
        } else {
            am[j] = rm[j] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = i + e < it.size;
                p[j][e] = in ? it.values[i + e] : 0.f;
                g[j][e] = in ? it.grad[i + e] : 0.f;
                if (in) {
                    am[j] |= (uint32_t)it.average[i + e] << (8 * e);
                    rm[j] |= (uint32_t)it.root[i + e] << (8 * e);
                }
            }
        }
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        const long long block = base / kBlock + b;
        const bool in = WHOLE || block * kBlock < it.size;
        a_scale[b] = in ? it.average_scale[block] : 0.f;
        r_scale[b] = in ? it.root_scale[block] : 0.f;
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        BlockScales scales;
        if (!WHOLE || !step_usual(p + 2 * b, g + 2 * b, am + 2 * b, rm + 2 * b, a_scale[b], r_scale[b], step, root_factor, rates, scales))
            scales = step_any(p + 2 * b, g + 2 * b, am + 2 * b, rm + 2 * b, a_scale[b], r_scale[b], step, root_factor, rates);
        if (lane == 0 && (WHOLE || (base / kBlock + b) * kBlock < it.size)) {
            it.average_scale[base / kBlock + b] = scales.m_scale;
            it.root_scale[base / kBlock + b] = scales.r_scale;
        }
    }
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
        const long long i = at(j);
        if (WHOLE) {
            *reinterpret_cast<float4*>(it.values + i) = *reinterpret_cast<const float4*>(p[j]);
            *reinterpret_cast<uint32_t*>(it.average + i) = am[j];
            *reinterpret_cast<uint32_t*>(it.root + i) = rm[j];
            if (it.shadow) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(p[j][0], p[j][1]), hi = __floats2bfloat162_rn(p[j][2], p[j][3]);
                *reinterpret_cast<uint2*>(it.shadow + i) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < it.size) {
                    it.values[i + e] = p[j][e];
                    it.average[i + e] = (uint8_t)(am[j] >> (8 * e));
                    it.root[i + e] = (uint8_t)(rm[j] >> (8 * e));
                    if (it.shadow) it.shadow[i + e] = __float2bfloat16_rn(p[j][e]);
                }
        }
    }
}

__device__ __forceinline__ bool aligned_item(const Item& it, bool step) {
    const uintptr_t wide = step ? (uintptr_t)it.values | (uintptr_t)it.grad : (uintptr_t)it.average_out | (uintptr_t)it.square_out;
    return (wide & 15u) == 0 && (((uintptr_t)it.average | (uintptr_t)it.root) & 3u) == 0 && (!step || ((uintptr_t)it.shadow & 7u) == 0);
}

// Items whose step's number the device keeps: one more, and the corrections that follow from it, a power to a thread.
template <bool FEW>
__global__ void __launch_bounds__(kThreads)
next_step_kernel(const __grid_constant__ FewItems few, const Item* __restrict__ table, int count, double learning_rate, double beta1, double beta2) {
    chain_begin();
    const Item* items = FEW ? few.item : table;
    for (int i = threadIdx.x; i < count; i += kThreads) {
        long long* kept = items[i].count;
        if (!kept || items[i].number) continue;
        const long long t = kept[0] + 1;
        kept[0] = t;
        *reinterpret_cast<float2*>(kept + 1) = make_float2((float)(learning_rate / (1 - pow(beta1, (double)t))), (float)(1 / sqrt(1 - pow(beta2, (double)t))));
    }
}

template <bool FEW>
__global__ void __launch_bounds__(kThreads)
adamw_bytes_kernel(const __grid_constant__ FewItems few, const Item* __restrict__ table, int count, long long total_chunks, Rates rates) {
    chain_begin();
    const Item* items = FEW ? few.item : table;
    Item it;
    long long last = 0;          // the item's chunks end here
    for (long long chunk = blockIdx.x; chunk < total_chunks; chunk += gridDim.x) {
        if (chunk >= last) {
            it = items[find_item(items, count, chunk)];
            last = it.first_chunk + (it.size + kChunk - 1) / kChunk;
            if (it.count && !it.number) {
                const float2 given = *reinterpret_cast<const float2*>(it.count + 1);
                it.step = given.x;
                it.root_factor = given.y;
            }
        }
        if (chunk == it.first_chunk && threadIdx.x == 0 && it.count && it.number) it.count[0] = it.number;
        const long long base = (chunk - it.first_chunk) * kChunk + (threadIdx.x >> 5) * (2 * kBlock);
        if (base >= it.size) continue;
        if (aligned_item(it, true) && base + 2 * kBlock <= it.size) step_blocks<true>(it, base, rates);
        else step_blocks<false>(it, base, rates);
    }
}

// what the codes stand for: average_out = m, square_out = r r
template <bool FEW>
__global__ void __launch_bounds__(kThreads)
byte_values_kernel(const __grid_constant__ FewItems few, const Item* __restrict__ table, int count, long long total_chunks) {
    chain_begin();
    const Item* items = FEW ? few.item : table;
    Item it;
    long long last = 0;
    bool vec = false;
    for (long long chunk = blockIdx.x; chunk < total_chunks; chunk += gridDim.x) {
        if (chunk >= last) {
            it = items[find_item(items, count, chunk)];
            last = it.first_chunk + (it.size + kChunk - 1) / kChunk;
            vec = aligned_item(it, false);
        }
        const long long base = (chunk - it.first_chunk) * kChunk + threadIdx.x * 4;
        uint32_t a[4], r[4];
        float as[4], rs[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const long long i = base + u * (kThreads * 4);
            a[u] = r[u] = 0;
            as[u] = rs[u] = 0.f;
            if (i >= it.size) continue;
            as[u] = it.average_scale[i / kBlock];
            rs[u] = it.root_scale[i / kBlock];
            if (vec && i + 4 <= it.size) {
                a[u] = *reinterpret_cast<const uint32_t*>(it.average + i);
                r[u] = *reinterpret_cast<const uint32_t*>(it.root + i);
            } else {
                for (int e = 0; e < 4 && i + e < it.size; ++e) {
                    a[u] |= (uint32_t)it.average[i + e] << (8 * e);
                    r[u] |= (uint32_t)it.root[i + e] << (8 * e);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const long long i = base + u * (kThreads * 4);
            if (i >= it.size) continue;
            float m[4], v[4];
            average_values(a[u], as[u], m);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float root = root_value((r[u] >> (8 * e)) & 255u, rs[u]);
                v[e] = __fmul_rn(root, root);
            }
            if (vec && i + 4 <= it.size) {
                *reinterpret_cast<float4*>(it.average_out + i) = make_float4(m[0], m[1], m[2], m[3]);
                *reinterpret_cast<float4*>(it.square_out + i) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < it.size) {
                        it.average_out[i + e] = m[e];
                        it.square_out[i + e] = v[e];
                    }
            }
        }
    }
}

// The numbers of all items lie apart from one another and from all codes and scales: in the order of their addresses nothing that is written reaches past the next start.
int values_apart(const qmoe_byte_item_t* items, int count) {
    struct Span { uint64_t at, end; bool written; };
    const std::unique_ptr<Span[]> spans(new (std::nothrow) Span[(size_t)count * 6]);
    if (!spans) { set_error("optimizer: no memory for a table of %d items", count); return QMOE_ERR_STATE; }
    Span* next = spans.get();
    for (int i = 0; i < count; ++i) {
        const qmoe_byte_item_t& it = items[i];
        const uint64_t n = (uint64_t)it.size, scales = (n + kBlock - 1) / kBlock * 4;
        for (const uint64_t at : {it.average_out, it.square_out}) *next++ = {at, at + n * 4, true};
        for (const uint64_t at : {it.average, it.root}) *next++ = {at, at + n, false};
        for (const uint64_t at : {it.average_scale, it.root_scale}) *next++ = {at, at + scales, false};
    }
    std::sort(spans.get(), next, [](const Span& a, const Span& b) { return a.at < b.at; });
    uint64_t written = 0, any = 0;          // where what came so far ends
    for (const Span* s = spans.get(); s != next; ++s) {
        if (s->at < written || (s->written && s->at < any)) return fail_arg("optimizer: an output overlaps another or what is read");
        if (s->written && s->end > written) written = s->end;
        if (s->end > any) any = s->end;
    }
    return 0;
}

// Validates the host's table and fills in first_chunk; a table of many items goes to `table` on the device.
// `counted`: some item's step has the number that follows from its count.
int stage(qmoe_byte_item_t* items, int count, uint64_t table, bool step, FewItems& few, long long* total, bool* counted, cudaStream_t stream) {
    if (!items || count <= 0) return fail_arg("optimizer: the item table is empty");
    if (count > kFewItems && (!table || (table & 15u))) return fail_arg("optimizer: the device table address must be non-null and 16-byte aligned");
    long long chunks = 0;
    bool given = false;
    *counted = false;
    for (int i = 0; i < count; ++i) {
        qmoe_byte_item_t& it = items[i];
        if (step && (it.count & 7u || it.number < 0)) return fail_arg("adamw: item %d has a misaligned count or a negative number", i);
        const bool follows = it.count && !it.number;
        given = given || !follows;
        *counted = *counted || follows;
        if (it.size <= 0) return fail_arg("optimizer: item %d has size %lld", i, (long long)it.size);
        if (!it.average || !it.average_scale || !it.root || !it.root_scale || (step ? !it.values || !it.grad : !it.average_out || !it.square_out))
            return fail_arg("optimizer: item %d has a null address", i);
        if ((it.values | it.grad | it.average_scale | it.root_scale | it.average_out | it.square_out) & 3u || it.shadow & 1u)
            return fail_arg("optimizer: item %d has a misaligned address", i);
        if (step && !follows && (!(it.step >= 0) || !(it.root_factor > 0) || isinf(it.step) || isinf(it.root_factor)))
            return fail_arg("adamw: item %d has a bias correction that is no positive number", i);
        it.first_chunk = chunks;
        chunks += (it.size + kChunk - 1) / kChunk;
    }
    *total = chunks;
    if (!step)
        if (int rc = values_apart(items, count)) return rc;
    if (step && given && qmoe_stream_capturing((uint64_t)stream))
        return fail_arg("adamw: a step whose number is given cannot be captured: a replay would take it again with the same bias corrections");
    if (count <= kFewItems) memcpy(few.item, items, (size_t)count * sizeof(Item));
    else if (qmoe_stream_capturing((uint64_t)stream)) return fail_arg("optimizer: more than %d items cannot be captured: a replay would copy the host's table as it is then", kFewItems);
    else QMOE_CUDA(cudaMemcpyAsync((void*)table, items, (size_t)count * sizeof(Item), cudaMemcpyHostToDevice, stream));
    return 0;
}

int grid_for(long long chunks) {
    const long long cap = (long long)sm_count() * 8;
    return (int)(chunks < cap ? chunks : cap);
}

}  // namespace
}  // namespace qmoe

using namespace qmoe;

extern "C" int64_t qmoe_byte_table_bytes(int32_t count) { return (int64_t)(count > 0 ? count : 0) * (int64_t)sizeof(qmoe_byte_item_t); }

extern "C" int qmoe_adamw_bytes(qmoe_byte_item_t* items, int32_t count, uint64_t table, double learning_rate, double beta1, double beta2, double eps,
                                double weight_decay, uint64_t stream_) {
    if (!(learning_rate >= 0) || !(eps >= 0) || !(weight_decay >= 0) || isinf(learning_rate) || isinf(eps) || isinf(weight_decay))
        return fail_arg("adamw: learning rate, eps and weight decay must be numbers that are not negative");
    if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1)) return fail_arg("adamw: betas must lie in [0, 1)");
    cudaStream_t stream = (cudaStream_t)stream_;
    FewItems few;
    long long chunks = 0;
    bool counted = false;
    if (int rc = stage(items, count, table, true, few, &chunks, &counted, stream)) return rc;
    TimedScope timed(KC_OPTIMIZER, stream);
    if (counted) {
        if (count <= kFewItems) chained(next_step_kernel<true>, 1, kThreads, 0, stream, few, nullptr, count, learning_rate, beta1, beta2);
        else chained(next_step_kernel<false>, 1, kThreads, 0, stream, few, (const Item*)table, count, learning_rate, beta1, beta2);
        QMOE_LAUNCH_CHECK("next_step_kernel");
    }
    const Rates rates = {(float)beta1, (float)(1 - beta1), (float)beta2, (float)(1 - beta2), (float)(1 - learning_rate * weight_decay), (float)eps * 0.0625f};
    if (count <= kFewItems) chained(adamw_bytes_kernel<true>, grid_for(chunks), kThreads, 0, stream, few, nullptr, count, chunks, rates);
    else chained(adamw_bytes_kernel<false>, grid_for(chunks), kThreads, 0, stream, few, (const Item*)table, count, chunks, rates);
    QMOE_LAUNCH_CHECK("adamw_bytes_kernel");
    return 0;
}

extern "C" int qmoe_byte_values(qmoe_byte_item_t* items, int32_t count, uint64_t table, uint64_t stream_) {
    cudaStream_t stream = (cudaStream_t)stream_;
    FewItems few;
    long long chunks = 0;
    bool counted = false;
    if (int rc = stage(items, count, table, false, few, &chunks, &counted, stream)) return rc;
    TimedScope timed(KC_OPTIMIZER, stream);
    if (count <= kFewItems) chained(byte_values_kernel<true>, grid_for(chunks), kThreads, 0, stream, few, nullptr, count, chunks);
    else chained(byte_values_kernel<false>, grid_for(chunks), kThreads, 0, stream, few, (const Item*)table, count, chunks);
    QMOE_LAUNCH_CHECK("byte_values_kernel");
    return 0;
}
