// The key/value cache of decoding: new positions written behind the ones a sequence holds, quantised to 8 bits on the way if the
// cache is an 8-bit one, and positions read back.  Both are streams: what bounds them is HBM, or the launch for a handful of rows.
//
// 8 bits are whole multiples of a scale of each head and position, max |x| / 127.  Against an 8-bit floating type under the same scale
// the error is a quarter (dim 64, normal values, by calculation: 0.7 % of the root mean square instead of 2.6 %), and the whole numbers are exact in
// bf16, so the attention that reads them can hand them to the tensor cores as they are.  The division is the rounded one
// of IEEE, not a product with the reciprocal: x / s then lies on the same side of a tie everywhere.
//
// dim / 16 lanes (rounded up to a power of two) hold a head of one position, 16 values each.
//
// Measured, 8 bits, 4 heads of 64: one position each of 64 sequences written and up to 301 of each read into bfloat16 9.7 us, 25 MB; 8192 positions written
// and read 9.6 us, 17 MB.  Two launches of which the second waits for the first are most of either; the division takes the append 60 % of the issue slots.
#include "common.cuh"

#include <type_traits>

namespace qmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;

// Values of a lane: 16, so that its 8-bit ones are one 16-byte access; 8 where the head width is no multiple of that
int lane_values(const qmoe_cache_t* c) { return c->dim % 16 ? 8 : 16; }

struct CacheParams {
    void* k;
    void* v;
    float* k_scale;
    float* v_scale;
    const int* lengths;
    long long capacity;
    unsigned units;                      // heads of positions, keys and values counted once
    int batch, kv_heads, dim, lane_bits;
    // append
    const void* k_in;
    const void* v_in;
    const int* counts;
    int* lengths_out;
    long long k_pitch, v_pitch;
    int time;
    // read
    void* k_read;
    void* v_read;
    long long start, count;
};

template <int V, typename T> __device__ __forceinline__ void load_values(const T* p, float* f) {
#pragma unroll
    for (int i = 0; i < V; i += Vec16<T>::N) Vec16<T>::unpack(*reinterpret_cast<const uint4*>(p + i), f + i);
}
template <int V, typename T> __device__ __forceinline__ void store_values(T* p, const float* f) {
#pragma unroll
    for (int i = 0; i < V; i += Vec16<T>::N) *reinterpret_cast<uint4*>(p + i) = Vec16<T>::pack(f + i);
}
__device__ __forceinline__ float max_or_nan(float a, float b) {      // a NaN among the values ends in the scale, not under the carpet
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// four values in -127 .. 127 as bytes
__device__ __forceinline__ uint32_t pack_bytes(const int* q) {
    return (uint32_t)(q[0] & 255) | (uint32_t)(q[1] & 255) << 8 | (uint32_t)(q[2] & 255) << 16 | (uint32_t)q[3] << 24;
}

template <int V> struct Bytes;           // V of them as one access
template <> struct Bytes<8> { using type = uint2; };
template <> struct Bytes<16> { using type = uint4; };

// Keys in blockIdx.y = 0, values in 1.  V values to a lane; a thread has its part of one head of one position.
template <typename T, bool INT8, int V>
__global__ void __launch_bounds__(kThreads)
cache_append_kernel(const __grid_constant__ CacheParams p) {
    chain_begin();
    const bool key = blockIdx.y == 0;
    const int lanes = 1 << p.lane_bits, sub = threadIdx.x & (lanes - 1);
    if (key)
        for (long long b = (long long)blockIdx.x * kThreads + threadIdx.x; b < p.batch; b += (long long)gridDim.x * kThreads) {
            const int n = p.counts ? min(max(p.counts[b], 0), p.time) : p.time;
            p.lengths_out[b] = (int)min(p.capacity, (long long)p.lengths[b] + n);
        }
    const unsigned unit = blockIdx.x * (kThreads >> p.lane_bits) + (threadIdx.x >> p.lane_bits);
    const bool in = unit < p.units;      // (the shuffles below need all of a warp's lanes)
    const unsigned row = in ? unit / (unsigned)p.kv_heads : 0, b = row / (unsigned)p.time;
    const int h = in ? (int)(unit - row * p.kv_heads) : 0, t = (int)(row - b * p.time);
    // the values are read whether they are wanted or not: nothing waits for the lengths but what is written
    const int held = p.lengths[b], wanted = p.counts ? min(p.counts[b], p.time) : p.time;
    float f[V] = {};
    if (in && sub * V < p.dim) load_values<V>((key ? (const T*)p.k_in + row * p.k_pitch : (const T*)p.v_in + row * p.v_pitch) + h * p.dim + V * sub, f);
    const long long position = (long long)held + t;
    const bool active = in && t < wanted && position >= 0 && position < p.capacity && sub * V < p.dim;
    const long long at = ((long long)b * p.kv_heads + h) * p.capacity + position;
    if constexpr (INT8) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) most = max_or_nan(most, fabsf(f[i]));
        for (int o = 1; o < lanes; o <<= 1) most = max_or_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float scale = __fdiv_rn(most, 127.f);
        if (!active) return;
        uint32_t words[V / 4];
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            int q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = scale > 0.f ? min(max(__float2int_rn(__fdiv_rn(f[i + e], scale)), -127), 127) : 0;
            words[i / 4] = pack_bytes(q);
        }
        *reinterpret_cast<typename Bytes<V>::type*>((int8_t*)(key ? p.k : p.v) + at * p.dim + V * sub) = *reinterpret_cast<const typename Bytes<V>::type*>(words);
        if (sub == 0) (key ? p.k_scale : p.v_scale)[at] = scale;
    } else if (active) {
        store_values<V>((__nv_bfloat16*)(key ? p.k : p.v) + at * p.dim + V * sub, f);
    }
}

template <typename T, bool INT8, int V>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const __grid_constant__ CacheParams p) {
    chain_begin();
    const bool key = blockIdx.y == 0;
    const int sub = threadIdx.x & ((1 << p.lane_bits) - 1);
    const unsigned unit = blockIdx.x * (kThreads >> p.lane_bits) + (threadIdx.x >> p.lane_bits);
    if (unit >= p.units || sub * V >= p.dim) return;
    const unsigned row = unit / (unsigned)p.kv_heads, b = row / (unsigned)p.count;
    const int h = (int)(unit - row * p.kv_heads);
    const long long position = p.start + (row - b * (unsigned)p.count);
    float f[V] = {};
    if (position < p.lengths[b] && position < p.capacity) {
        const long long at = ((long long)b * p.kv_heads + h) * p.capacity + position;
        if constexpr (INT8) {
            const typename Bytes<V>::type raw = *reinterpret_cast<const typename Bytes<V>::type*>((const int8_t*)(key ? p.k : p.v) + at * p.dim + V * sub);
            const float scale = (key ? p.k_scale : p.v_scale)[at];
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * scale;
        } else {
            load_values<V>((const __nv_bfloat16*)(key ? p.k : p.v) + at * p.dim + V * sub, f);
        }
    }
    store_values<V>((T*)(key ? p.k_read : p.v_read) + ((long long)row * p.kv_heads + h) * p.dim + V * sub, f);
}

CacheParams cache_params(const qmoe_cache_t* c) {
    CacheParams p = {};
    p.k = (void*)c->k; p.v = (void*)c->v; p.k_scale = (float*)c->k_scale; p.v_scale = (float*)c->v_scale;
    p.lengths = (const int*)c->lengths;
    p.capacity = c->capacity; p.batch = (int)c->batch; p.kv_heads = c->kv_heads; p.dim = c->dim;
    while ((lane_values(c) << p.lane_bits) < c->dim) ++p.lane_bits;
    return p;
}

template <bool APPEND> int launch(CacheParams& p, const qmoe_cache_t* c, long long positions, int dtype, cudaStream_t stream) {
    // (the kernels number the heads of positions in 32 bits, with a block's worth of room behind the last)
    if (positions > 0x7fffffffll / c->batch || positions * c->batch > 0x7fffffffll / c->kv_heads)
        return fail_arg("cache: more than 2147483647 heads of positions in one call");
    const long long units = c->batch * positions * c->kv_heads;
    p.units = (unsigned)units;
    const dim3 grid((unsigned)ceil_div(units, kThreads >> p.lane_bits), 2);
    auto go = [&](auto value, auto int8, auto values) {
        using T = decltype(value);
        if constexpr (APPEND) chained(cache_append_kernel<T, decltype(int8)::value, decltype(values)::value>, grid, kThreads, 0, stream, p);
        else chained(cache_read_kernel<T, decltype(int8)::value, decltype(values)::value>, grid, kThreads, 0, stream, p);
    };
    auto by_width = [&](auto value, auto int8) {
        if (lane_values(c) == 16) go(value, int8, std::integral_constant<int, 16>());
        else go(value, int8, std::integral_constant<int, 8>());
    };
    auto by_cache = [&](auto value) {
        if (c->dtype == QMOE_INT8) by_width(value, std::true_type());
        else by_width(value, std::false_type());
    };
    if (dtype == QMOE_BF16) by_cache(__nv_bfloat16());
    else by_cache(float());
    QMOE_LAUNCH_CHECK(APPEND ? "cache_append_kernel" : "cache_read_kernel");
    return 0;
}

}  // namespace

int cache_check(const qmoe_cache_t* c) {
    if (!c) return fail_arg("cache is null");
    if (c->batch <= 0 || c->capacity <= 0 || c->kv_heads <= 0 || c->batch > 0x7fffffff || c->capacity > 0x7fffffff)
        return fail_arg("cache: batch, capacity and kv_heads must be positive 32-bit numbers");
    if (c->dim < 8 || c->dim > kMaxDim || c->dim % 8) return fail_arg("cache: the head width must be a multiple of 8 up to %d", kMaxDim);
    if (c->dtype != QMOE_BF16 && c->dtype != QMOE_INT8) return fail_arg("cache: dtype must be QMOE_BF16 or QMOE_INT8");
    if (!c->k || !c->v || !c->lengths) return fail_arg("cache: null buffer address");
    if (c->dtype == QMOE_INT8 && (!c->k_scale || !c->v_scale)) return fail_arg("cache: an 8-bit cache needs its scales");
    if ((c->k | c->v) & 15u || (c->k_scale | c->v_scale | c->lengths) & 3u) return fail_arg("cache: buffers must be 16-byte aligned, scales and lengths 4-byte");
    return 0;
}

}  // namespace qmoe

using namespace qmoe;

extern "C" int qmoe_cache_append(const qmoe_cache_t* c, uint64_t k, uint64_t v, int32_t dtype, int64_t k_pitch, int64_t v_pitch, int64_t time,
                                 uint64_t counts, uint64_t lengths_out, uint64_t stream_) {
    if (int rc = cache_check(c)) return rc;
    if (dtype != QMOE_F32 && dtype != QMOE_BF16) return fail_arg("cache_append: dtype must be QMOE_F32 or QMOE_BF16");
    if (time < 0 || time > c->capacity) return fail_arg("cache_append: time must lie between 0 and the capacity");
    if (!lengths_out || lengths_out & 3u || counts & 3u) return fail_arg("cache_append: null or misaligned lengths");
    // blocks read the old lengths and the counts while others write the new lengths
    auto overlaps = [&](uint64_t read) { return read && read < lengths_out + c->batch * sizeof(int) && lengths_out < read + c->batch * sizeof(int); };
    if (overlaps(c->lengths) || overlaps(counts)) return fail_arg("cache_append: the new lengths need a buffer of their own");
    cudaStream_t stream = (cudaStream_t)stream_;
    if (!time) {
        QMOE_CUDA(cudaMemcpyAsync((void*)lengths_out, (const void*)c->lengths, c->batch * sizeof(int), cudaMemcpyDeviceToDevice, stream));
        return 0;
    }
    const long long align = dtype == QMOE_BF16 ? 8 : 4, width = (long long)c->kv_heads * c->dim;
    if (!k || !v || (k | v) & 15u) return fail_arg("cache_append: k and v must be non-null and 16-byte aligned");
    if (k_pitch < width || v_pitch < width || k_pitch % align || v_pitch % align)
        return fail_arg("cache_append: a row pitch must be a multiple of 16 bytes and not below the row's width");
    TimedScope timed(KC_ELEMENTWISE, stream);
    CacheParams p = cache_params(c);
    p.k_in = (const void*)k; p.v_in = (const void*)v; p.k_pitch = k_pitch; p.v_pitch = v_pitch;
    p.counts = (const int*)counts; p.lengths_out = (int*)lengths_out; p.time = (int)time;
    return launch<true>(p, c, time, dtype, stream);
}

extern "C" int qmoe_cache_read(const qmoe_cache_t* c, int64_t start, int64_t count, uint64_t k_out, uint64_t v_out, int32_t dtype, uint64_t stream_) {
    if (int rc = cache_check(c)) return rc;
    if (dtype != QMOE_F32 && dtype != QMOE_BF16) return fail_arg("cache_read: dtype must be QMOE_F32 or QMOE_BF16");
    if (start < 0 || count < 0 || start > c->capacity || count > c->capacity - start) return fail_arg("cache_read: positions outside the cache");
    if (!count) return 0;
    if (!k_out || !v_out || (k_out | v_out) & 15u) return fail_arg("cache_read: outputs must be non-null and 16-byte aligned");
    cudaStream_t stream = (cudaStream_t)stream_;
    TimedScope timed(KC_ELEMENTWISE, stream);
    CacheParams p = cache_params(c);
    p.k_read = (void*)k_out; p.v_read = (void*)v_out; p.start = start; p.count = count;
    return launch<false>(p, c, count, dtype, stream);
}
