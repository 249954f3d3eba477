// The norm of every query and key head and the rotation of its position, queries and keys in one pass:
//     y = R(p) (w * x / rms(x)),   rms(x) = sqrt(mean(x^2) + eps) over the head's `dim` elements,
// with R(p) turning every pair (2 i, 2 i + 1) by the angle p theta^(-2 i / dim), p the row's position.  Backward, from g = dL/dy:
//     g' = R(-p) g,   dw = sum over rows and heads of g' * x / rms,   dx = (g' * w - x / rms * mean(g' * w * x / rms)) / rms.
// The statistics are not kept from the forward: a head is in a few lanes' registers anyway.
//
// dim / 8 lanes (rounded up to a power of two) hold a head, eight elements each, so a warp has 32 / lanes heads at a time, and
// goes through a chunk of a row's heads.  The row's angles are formed once, a pair to a lane, and handed on through shared memory.
//
// Angles.  A position times a frequency is a place on the circle, and what counts is its fraction of a turn: the frequency in
// turns is held as a 64-bit fraction F (2^64 = one turn), so position * F modulo 2^64, an integer product, IS that fraction for F, and its upper half
// goes to sincospi.  F itself comes from a running product of up to 128 rounded factors, off by at most 2^-58 turns for theta from 1 on, so the angle of
// position p is exact to 2^-58 p turns.  (In 32 bits the angle of position 100000 is off by 4e-3.)
// Sums over rows run in a fixed order (no atomics).
//
// What bounds it: the instructions, issued in 68 % of the cycles forward and 63 % backward.  8192 rows of 16 and 4 heads of 64 in bfloat16: forward
// 11.5 us, 42 MB at 3.6 TB/s; backward 18 us, 63 MB at 3.5 TB/s, and 5 us for the joined sum of its blocks' shares of the weights' gradients.
#include "common.cuh"

#include <math.h>
#include <stddef.h>
#include <string.h>

#include <type_traits>

namespace qmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 256;
constexpr int kInFlight = 4;             // heads of a lane whose loads are on their way together

struct NormRopeParams {
    const void* q;
    const void* k;
    void* q_out;                         // backward: dq, dk
    void* k_out;
    const void* grad_q;
    const void* grad_k;
    const float* q_weight;
    const float* k_weight;
    const int* starts;
    float* partials;
    long long offset, q_pitch, k_pitch;
    int rows, time, heads, kv_heads, dim;
    int lane_bits, all_passes, passes;   // log2 of the lanes per head; passes of a row, of a chunk of it
    float eps, one_over_dim;
    unsigned long long turns[kMaxDim / 2];
};

__device__ __forceinline__ void load8(const __nv_bfloat16* p, uint4* raw) { raw[0] = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void load8(const float* p, uint4* raw) {
    raw[0] = *reinterpret_cast<const uint4*>(p);
    raw[1] = *reinterpret_cast<const uint4*>(p + 4);
}
template <typename T> __device__ __forceinline__ void unpack8(const uint4* raw, float* f) {
    Vec16<T>::unpack(raw[0], f);
    if constexpr (Vec16<T>::N == 4) Vec16<T>::unpack(raw[1], f + 4);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* f) {
    *reinterpret_cast<uint4*>(p) = Vec16<T>::pack(f);
    if constexpr (Vec16<T>::N == 4) *reinterpret_cast<uint4*>(p + 4) = Vec16<T>::pack(f + 4);
}
// sum over the 2^bits neighbouring lanes of a head, in every one of them
template <int BITS> __device__ __forceinline__ float head_sum(float v, int bits) {
    if constexpr (BITS >= 0) {
#pragma unroll
        for (int o = 1; o < 1 << BITS; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    } else {
        for (int o = 1; o < 1 << bits; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

// What a warp of a block has: its lanes' place in a head, the weights of query and key heads and the angles of its row in shared memory.  The
// row's heads go by in passes of `per_warp` heads, the query heads' passes first, the key heads' behind them.
template <typename T> struct Warp {
    const NormRopeParams& p;
    float2* angles;                      // cosine and sine of the row's dim / 2 angles
    const float* weights;                // [query, key][dim]
    const unsigned long long* turns;
    int sub, slot, per_warp, query_passes;
    bool active;
    __device__ __forceinline__ Warp(const NormRopeParams& p_, float2 (*s_angles)[kMaxDim / 2], float* s_weights) : p(p_) {
        const int lane = threadIdx.x & 31;
        angles = s_angles[threadIdx.x >> 5];
        weights = s_weights;
        sub = lane & ((1 << p.lane_bits) - 1);
        slot = lane >> p.lane_bits;
        per_warp = 32 >> p.lane_bits;
        query_passes = (p.heads + per_warp - 1) >> (5 - p.lane_bits);
        active = sub * 8 < p.dim;
    }
    // the block's weights and frequencies into shared memory; the first rows' loads are on their way by then
    __device__ __forceinline__ void stage(float* s_weights, unsigned long long* s_turns) {
        for (int i = threadIdx.x; i < 2 * p.dim; i += kThreads) s_weights[i] = i < p.dim ? p.q_weight[i] : p.k_weight[i - p.dim];
        // (a parameter's element by the lane's number is a load for each lane)
        for (int i = threadIdx.x; i < p.dim / 2; i += kThreads) s_turns[i] = p.turns[i];
        turns = s_turns;
        __syncthreads();
    }
    // a lane's part of its head in a pass, or -1
    __device__ __forceinline__ int head(int pass) const {
        const int h = (pass < query_passes ? pass : pass - query_passes) * per_warp + slot;
        return active && h < (pass < query_passes ? p.heads : p.kv_heads) ? h : -1;
    }
    // every pair once in the warp, and from there to the lanes of all heads
    __device__ __forceinline__ void turn(int row) const {
        const int b = row / p.time;
        const long long position = p.offset + (p.starts ? p.starts[b] : 0) + (row - b * p.time);
        __syncwarp();                    // the row before is done with them
        for (int i = threadIdx.x & 31; i < p.dim / 2; i += 32) {
            const int turned = (int)(((unsigned long long)position * turns[i]) >> 32);       // of 2^32
            float2 v;
            sincospif((float)turned * 4.656612873077392578125e-10f, &v.y, &v.x);              // 2^-31: half turns
            angles[i] = v;
        }
        __syncwarp();
    }
    __device__ __forceinline__ void angle(float* c, float* s) const {
        const float4* from = reinterpret_cast<const float4*>(angles + (active ? 4 * sub : 0));
        const float4 a = from[0], b = from[1];
        c[0] = a.x; s[0] = a.y; c[1] = a.z; s[1] = a.w;
        c[2] = b.x; s[2] = b.y; c[3] = b.z; s[3] = b.w;
    }
    __device__ __forceinline__ void weight(int pass, float* w) const {
        const float4* from = reinterpret_cast<const float4*>(weights + (pass < query_passes ? 0 : p.dim) + (active ? 8 * sub : 0));
        const float4 a = from[0], b = from[1];
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    // Where this lane's part of the first query and key head of a row lies: in rows `pitch` elements apart, and densely
    struct Row { long long q, k; };
    __device__ __forceinline__ Row pitched(int row) const { return {row * p.q_pitch + slot * p.dim + 8 * sub, row * p.k_pitch + slot * p.dim + 8 * sub}; }
    __device__ __forceinline__ Row dense(int row) const {
        return {(long long)row * (p.heads * p.dim) + slot * p.dim + 8 * sub, (long long)row * (p.kv_heads * p.dim) + slot * p.dim + 8 * sub};
    }
    template <typename P> __device__ __forceinline__ P* at(P* q, P* k, const Row& row, int pass) const {
        const bool query = pass < query_passes;
        return (query ? q : k) + ((query ? row.q : row.k) + (query ? pass : pass - query_passes) * per_warp * p.dim);
    }
};

// a row's chunk of heads to a warp
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads, 4)
norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
    chain_begin();
    __shared__ __align__(16) float2 s_angles[kWarps][kMaxDim / 2];
    __shared__ __align__(16) float s_weights[2 * kMaxDim];
    __shared__ unsigned long long s_turns[kMaxDim / 2];
    Warp<T> me(p, s_angles, s_weights);
    const int row = blockIdx.x * kWarps + (threadIdx.x >> 5), last = row < p.rows ? min(p.all_passes, (int)(blockIdx.y + 1) * p.passes) : 0;
    const auto from = me.pitched(row), to = me.dense(row);
    uint4 raw[kInFlight][2];
    auto fetch = [&](int at) {
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
            if (at + u < last && me.head(at + u) >= 0) load8(me.at((const T*)p.q, (const T*)p.k, from, at + u), raw[u]);
            else raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
        }
    };
    int at = blockIdx.y * p.passes;
    fetch(at);
    me.stage(s_weights, s_turns);
    if (at >= last) return;
    float s[4], c[4];
    me.turn(row);
    me.angle(c, s);
    while (true) {
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
            if (at + u >= last) break;
            const int h = me.head(at + u);
            float x[8], y[8], w[8], square = 0.f;
            unpack8<T>(raw[u], x);
#pragma unroll
            for (int i = 0; i < 8; ++i) square = fmaf(x[i], x[i], square);
            const float inverse = rsqrtf(head_sum<BITS>(square, p.lane_bits) * p.one_over_dim + p.eps);
            me.weight(at + u, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = x[2 * i] * w[2 * i], b = x[2 * i + 1] * w[2 * i + 1], ci = c[i] * inverse, si = s[i] * inverse;
                y[2 * i] = a * ci - b * si;
                y[2 * i + 1] = a * si + b * ci;
            }
            if (h >= 0) store8(me.at((T*)p.q_out, (T*)p.k_out, to, at + u), y);
        }
        at += kInFlight;
        if (at >= last) return;
        fetch(at);
    }
}

// dq, dk, and this block's share of the weights' gradients: partials[block][q | k][dim]
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads, 3)
norm_rope_backward_kernel(const __grid_constant__ NormRopeParams p) {
    chain_begin();
    constexpr int TOGETHER = kInFlight / 2;
    __shared__ __align__(16) float2 s_angles[kWarps][kMaxDim / 2];
    __shared__ __align__(16) float s_weights[2 * kMaxDim];
    __shared__ float s_sum[kWarps][2][kMaxDim];
    __shared__ unsigned long long s_turns[kMaxDim / 2];
    Warp<T> me(p, s_angles, s_weights);
    me.stage(s_weights, s_turns);
    const int first = blockIdx.y * p.passes, last = min(p.all_passes, first + p.passes);
    float dwq[8] = {}, dwk[8] = {};
    for (int row = blockIdx.x * kWarps + (threadIdx.x >> 5); row < p.rows; row += gridDim.x * kWarps) {
        const auto from = me.pitched(row), to = me.dense(row);
        float s[4], c[4];
        bool turned = false;
        for (int at = first; at < last; at += TOGETHER) {
            uint4 raw[TOGETHER][2], raw_g[TOGETHER][2];
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u) {
                const int h = at + u < last ? me.head(at + u) : -1;
                if (h >= 0) {
                    load8(me.at((const T*)p.q, (const T*)p.k, from, at + u), raw[u]);
                    load8(me.at((const T*)p.grad_q, (const T*)p.grad_k, to, at + u), raw_g[u]);
                } else {
                    raw[u][0] = raw[u][1] = raw_g[u][0] = raw_g[u][1] = make_uint4(0, 0, 0, 0);
                }
            }
            if (!turned) {
                me.turn(row);
                me.angle(c, s);
                turned = true;
            }
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u) {
                if (at + u >= last) break;
                const int h = me.head(at + u);
                float x[8], g[8], w[8], square = 0.f, dot = 0.f;
                unpack8<T>(raw[u], x);
                unpack8<T>(raw_g[u], g);
#pragma unroll
                for (int i = 0; i < 8; ++i) square = fmaf(x[i], x[i], square);
                const float mean = head_sum<BITS>(square, p.lane_bits) * p.one_over_dim + p.eps;
                const float inverse = h >= 0 ? rsqrtf(mean) : 0.f;       // a place without a head has zeros, and 0 / sqrt(0) were eps zero
                me.weight(at + u, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) {          // turned back
                    const float a = g[2 * i], b = g[2 * i + 1];
                    g[2 * i] = a * c[i] + b * s[i];
                    g[2 * i + 1] = b * c[i] - a * s[i];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= inverse;
                // zero where there is no head
                if (at + u < me.query_passes) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) dwq[i] = fmaf(g[i], x[i], dwq[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) dwk[i] = fmaf(g[i], x[i], dwk[i]);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    g[i] *= w[i];
                    dot = fmaf(g[i], x[i], dot);
                }
                dot = head_sum<BITS>(dot, p.lane_bits) * p.one_over_dim;
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = inverse * (g[i] - x[i] * dot);
                if (h >= 0) store8(me.at((T*)p.q_out, (T*)p.k_out, to, at + u), g);
            }
        }
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        for (int o = 1 << p.lane_bits; o < 32; o <<= 1) {
            dwq[i] += __shfl_xor_sync(0xffffffffu, dwq[i], o);
            dwk[i] += __shfl_xor_sync(0xffffffffu, dwk[i], o);
        }
        if (lane < 1 << p.lane_bits) {
            s_sum[warp][0][8 * me.sub + i] = dwq[i];
            s_sum[warp][1][8 * me.sub + i] = dwk[i];
        }
    }
    __syncthreads();
    float* out = p.partials + (long long)(blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.dim;
    for (int j = threadIdx.x; j < 2 * p.dim; j += kThreads) {
        const int which = j >= p.dim, column = j - which * p.dim;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += s_sum[w][which][column];
        out[j] = sum;
    }
}

// 32 columns of the weights' gradients to a block: its 32 warps stride over the blocks' shares, all of a warp's loads in flight together, and meet
// in a fixed order
constexpr int kWeightThreads = 1024, kShares = 16;
__global__ void __launch_bounds__(kWeightThreads)
norm_rope_weights_kernel(const float* __restrict__ partials, float* __restrict__ dq_weight, float* __restrict__ dk_weight, int blocks, int dim) {
    chain_begin();
    __shared__ float s_sum[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, column = blockIdx.x * 32 + lane;
    float sum = 0.f;
    for (int b = warp; b < blocks; b += 32 * kShares) {
        float v[kShares];
#pragma unroll
        for (int i = 0; i < kShares; ++i) v[i] = b + 32 * i < blocks && column < 2 * dim ? partials[(long long)(b + 32 * i) * 2 * dim + column] : 0.f;
#pragma unroll
        for (int i = 0; i < kShares; ++i) sum += v[i];
    }
    s_sum[warp][lane] = sum;
    __syncthreads();
    sum = warp_sum(s_sum[lane][warp]);               // warp: a column now
    const int mine = blockIdx.x * 32 + warp;
    if (lane == 0 && mine < 2 * dim) (mine < dim ? dq_weight : dk_weight - dim)[mine] = sum;
}

struct Shape { int lane_bits, all_passes, passes, chunks, blocks; };

// Lanes per head, and how a row's passes are cut into chunks: whole rows to a warp (angles formed once) while the rows alone make
// eight warps per SM, else shorter chunks down to one pass.  `blocks`: of eight rows; for the backward at most three to an SM, which walk the rows
// and leave one share of the weights' gradients each.
Shape shape_of(long long rows, int heads, int kv_heads, int dim, bool backward) {
    Shape s = {};
    while ((8 << s.lane_bits) < dim) ++s.lane_bits;
    const int per_warp = 32 >> s.lane_bits;
    s.all_passes = s.passes = ceil_div(heads, per_warp) + ceil_div(kv_heads, per_warp);
    while (s.passes > 1 && rows * ceil_div(s.all_passes, s.passes) < (long long)sm_count() * 8) s.passes = (s.passes + 1) / 2;
    s.chunks = ceil_div(s.all_passes, s.passes);
    s.blocks = ceil_div(rows, kWarps);
    if (backward) {
        const int most = 3 * sm_count() / s.chunks > 1 ? 3 * sm_count() / s.chunks : 1;
        if (s.blocks > most) s.blocks = most;
    }
    return s;
}

// the usual widths with their lanes known to the compiler, others with a loop (8192 rows of 16 and 4 heads of 64, both directions: 34.8 us and 36.8)
template <typename Launch> void launch_by_width(const qmoe_norm_rope_t* a, Launch launch) {
    auto by_type = [&](auto value) {
        if (a->dim == 64) launch(value, std::integral_constant<int, 3>());
        else if (a->dim == 128) launch(value, std::integral_constant<int, 4>());
        else launch(value, std::integral_constant<int, -1>());
    };
    if (a->dtype == QMOE_BF16) by_type(__nv_bfloat16());
    else by_type(float());
}

int norm_rope_check(const qmoe_norm_rope_t* a, bool backward) {
    if (!a) return fail_arg("norm_rope: argument is null");
    if (a->dtype != QMOE_F32 && a->dtype != QMOE_BF16) return fail_arg("norm_rope: dtype must be QMOE_F32 or QMOE_BF16");
    if (a->batch < 0 || a->time < 0 || a->heads <= 0 || a->kv_heads <= 0) return fail_arg("norm_rope: sizes must not be negative, head counts positive");
    if (a->dim < 8 || a->dim > kMaxDim || a->dim % 8) return fail_arg("norm_rope: the head width must be a multiple of 8 up to %d", kMaxDim);
    if (a->heads > (1 << 20) || a->kv_heads > (1 << 20) || (a->batch && a->time > 0x7fffffff / a->batch)) return fail_arg("norm_rope: too many rows or heads");
    if (!(a->theta > 0) || !(a->eps >= 0) || a->theta > 1e30) return fail_arg("norm_rope: theta must be positive and eps not negative");
    if (!a->q || !a->k || !a->q_weight || !a->k_weight) return fail_arg("norm_rope: null buffer address");
    if (backward ? !a->grad_q || !a->grad_k || !a->dq || !a->dk || !a->d_q_weight || !a->d_k_weight || !a->partials : !a->q_out || !a->k_out)
        return fail_arg("norm_rope: null buffer address");
    if ((a->q | a->k | a->q_out | a->k_out | a->grad_q | a->grad_k | a->dq | a->dk) & 15u) return fail_arg("norm_rope: rows must be 16-byte aligned");
    if ((a->q_weight | a->k_weight | a->starts | a->partials | a->d_q_weight | a->d_k_weight) & 3u) return fail_arg("norm_rope: misaligned address");
    const long long align = a->dtype == QMOE_BF16 ? 8 : 4;
    if (a->q_pitch % align || a->k_pitch % align || a->q_pitch < (long long)a->heads * a->dim || a->k_pitch < (long long)a->kv_heads * a->dim)
        return fail_arg("norm_rope: a row pitch must be a multiple of 16 bytes and not below the row's width");
    // A lane writes where it has read or somewhere else altogether: rows of another pitch, or of the other heads, would be written before they are read
    struct Span { uint64_t at, bytes; };
    const uint64_t item = a->dtype == QMOE_BF16 ? 2 : 4, rows = (uint64_t)a->batch * (uint64_t)a->time;
    const uint64_t widths[2] = {(uint64_t)a->heads * a->dim, (uint64_t)a->kv_heads * a->dim}, pitches[2] = {(uint64_t)a->q_pitch, (uint64_t)a->k_pitch};
    const uint64_t in[2] = {a->q, a->k}, grad[2] = {a->grad_q, a->grad_k}, out[2] = {backward ? a->dq : a->q_out, backward ? a->dk : a->k_out};
    auto dense = [&](const uint64_t* of, int i) { return Span{of[i], rows * widths[i] * item}; };
    auto overlap = [](const Span& x, const Span& y) { return x.at < y.at + y.bytes && y.at < x.at + x.bytes; };
    bool apart = !rows || !overlap(dense(out, 0), dense(out, 1));
    for (int i = 0; rows && i < 2; ++i)
        for (int j = 0; j < 2; ++j) {
            const Span read = {in[j], ((rows - 1) * pitches[j] + widths[j]) * item};
            apart = apart && ((i == j && out[i] == in[j] && pitches[j] == widths[j]) || !overlap(dense(out, i), read));
            if (backward) apart = apart && ((i == j && out[i] == grad[j]) || !overlap(dense(out, i), dense(grad, j)));
        }
    if (!apart) return fail_arg("norm_rope: an output may lie on its own operand, row on row, and on no other");
    return 0;
}

void norm_rope_params(const qmoe_norm_rope_t* a, const Shape& s, NormRopeParams& p) {
    p.q = (const void*)a->q; p.k = (const void*)a->k;
    p.q_weight = (const float*)a->q_weight; p.k_weight = (const float*)a->k_weight;
    p.starts = (const int*)a->starts;
    p.offset = a->offset; p.q_pitch = a->q_pitch; p.k_pitch = a->k_pitch;
    p.rows = (int)(a->batch * a->time); p.time = (int)a->time;
    p.heads = a->heads; p.kv_heads = a->kv_heads; p.dim = a->dim;
    p.lane_bits = s.lane_bits; p.all_passes = s.all_passes; p.passes = s.passes;
    p.eps = (float)a->eps; p.one_over_dim = 1.f / a->dim;
    // the frequencies depend on theta and the width alone: a program has one of each (1.5 us a call where they are formed every time)
    static thread_local struct { double theta; int dim; unsigned long long turns[kMaxDim / 2]; } made = {};
    if (made.theta != a->theta || made.dim != a->dim) {
        const long double ratio = powl((long double)a->theta, -2.0L / a->dim);
        long double turns = 1.0L / 6.283185307179586476925286766559L;
        for (int i = 0; i < a->dim / 2; ++i, turns *= ratio) {
            const long double fraction = ldexpl(turns - floorl(turns), 64);
            made.turns[i] = fraction >= 18446744073709551615.0L ? 0ull : (unsigned long long)fraction;
        }
        made.theta = a->theta;
        made.dim = a->dim;
    }
    memcpy(p.turns, made.turns, a->dim / 2 * sizeof(p.turns[0]));
}

}  // namespace
}  // namespace qmoe

using namespace qmoe;

extern "C" int qmoe_norm_rope_forward(const qmoe_norm_rope_t* a, uint64_t stream_) {
    if (int rc = norm_rope_check(a, false)) return rc;
    if (!a->batch || !a->time) return 0;
    cudaStream_t stream = (cudaStream_t)stream_;
    TimedScope timed(KC_ELEMENTWISE, stream);
    const Shape s = shape_of(a->batch * a->time, a->heads, a->kv_heads, a->dim, false);
    NormRopeParams p;
    memset(&p, 0, offsetof(NormRopeParams, turns));
    norm_rope_params(a, s, p);
    p.q_out = (void*)a->q_out; p.k_out = (void*)a->k_out;
    const dim3 grid((unsigned)s.blocks, (unsigned)s.chunks);
    launch_by_width(a, [&](auto value, auto bits) { chained(norm_rope_kernel<decltype(value), decltype(bits)::value>, grid, kThreads, 0, stream, p); });
    QMOE_LAUNCH_CHECK("norm_rope_kernel");
    return 0;
}

extern "C" int64_t qmoe_norm_rope_partials(int64_t batch, int64_t time, int32_t heads, int32_t kv_heads, int32_t dim) {
    if (batch <= 0 || time <= 0 || heads <= 0 || kv_heads <= 0 || dim < 8 || dim > kMaxDim) return 1;
    const Shape s = shape_of(batch * time, heads, kv_heads, dim, true);
    return (int64_t)s.blocks * s.chunks * 2 * dim;
}

extern "C" int qmoe_norm_rope_backward(const qmoe_norm_rope_t* a, uint64_t stream_) {
    if (int rc = norm_rope_check(a, true)) return rc;
    cudaStream_t stream = (cudaStream_t)stream_;
    TimedScope timed(KC_ELEMENTWISE, stream);
    if (!a->batch || !a->time) {       // no rows: nothing but the weights' gradients to write
        QMOE_CUDA(cudaMemsetAsync((void*)a->d_q_weight, 0, a->dim * sizeof(float), stream));
        QMOE_CUDA(cudaMemsetAsync((void*)a->d_k_weight, 0, a->dim * sizeof(float), stream));
        return 0;
    }
    const Shape s = shape_of(a->batch * a->time, a->heads, a->kv_heads, a->dim, true);
    NormRopeParams p;
    memset(&p, 0, offsetof(NormRopeParams, turns));
    norm_rope_params(a, s, p);
    p.q_out = (void*)a->dq; p.k_out = (void*)a->dk;
    p.grad_q = (const void*)a->grad_q; p.grad_k = (const void*)a->grad_k;
    p.partials = (float*)a->partials;
    const dim3 grid((unsigned)s.blocks, (unsigned)s.chunks);
    launch_by_width(a, [&](auto value, auto bits) { chained(norm_rope_backward_kernel<decltype(value), decltype(bits)::value>, grid, kThreads, 0, stream, p); });
    QMOE_LAUNCH_CHECK("norm_rope_backward_kernel");
    chained(norm_rope_weights_kernel, (unsigned)ceil_div(2 * a->dim, 32), kWeightThreads, 0, stream, (const float*)a->partials, (float*)a->d_q_weight,
            (float*)a->d_k_weight, s.blocks * s.chunks, a->dim);
    QMOE_LAUNCH_CHECK("norm_rope_weights_kernel");
    return 0;
}
