// The key/value cache of decoding: new positions written behind the ones a sequence holds, quantised to 8 bits on the way if the
// cache is an 8-bit one, and positions read back.  Both are streams: what bounds them is HBM, or the launch for a handful of rows.
//
// 8 bits are whole multiples of a scale of each head and position, max |x| / 127.  Against an 8-bit floating type under the same scale
// the error is a quarter (dim 64, normal values: 0.7 % of the root mean square instead of 2.6 %), and the whole numbers are exact in
// bf16, so the attention that reads them can hand them to the tensor cores as they are.  The division is the rounded one
// of IEEE, not a product with the reciprocal: x / s then lies on the same side of a tie everywhere.
//
// dim / 8 lanes (rounded up to a power of two) hold a head of one position, eight values each.
#include "common.cuh"

namespace qmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;

struct CacheParams {
    void* k;
    void* v;
    float* k_scale;
    float* v_scale;
    const int* lengths;
    long long capacity, units;           // units: heads of positions, keys and values counted once
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

template <typename T> __device__ __forceinline__ void load_values(const T* p, float* f) {
#pragma unroll
    for (int i = 0; i < 8; i += Vec16<T>::N) Vec16<T>::unpack(*reinterpret_cast<const uint4*>(p + i), f + i);
}
template <typename T> __device__ __forceinline__ void store_values(T* p, const float* f) {
#pragma unroll
    for (int i = 0; i < 8; i += Vec16<T>::N) *reinterpret_cast<uint4*>(p + i) = Vec16<T>::pack(f + i);
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

// Keys in blockIdx.y = 0, values in 1.
template <typename T, bool INT8>
__global__ void __launch_bounds__(kThreads)
cache_append_kernel(const __grid_constant__ CacheParams p) {
    chain_begin();
    const bool key = blockIdx.y == 0;
    const int lanes = 1 << p.lane_bits, sub = threadIdx.x & (lanes - 1);
    const long long stride = (long long)gridDim.x * (kThreads >> p.lane_bits);
    if (key)
        for (long long b = (long long)blockIdx.x * kThreads + threadIdx.x; b < p.batch; b += (long long)gridDim.x * kThreads) {
            const int n = p.counts ? min(max(p.counts[b], 0), p.time) : p.time;
            p.lengths_out[b] = (int)min(p.capacity, (long long)p.lengths[b] + n);
        }
    // a warp's lanes go round together: the shuffles below need all of them
    for (long long unit = (long long)blockIdx.x * (kThreads >> p.lane_bits) + (threadIdx.x >> p.lane_bits);
         __any_sync(0xffffffffu, unit < p.units); unit += stride) {
        const bool in = unit < p.units;
        const long long row = in ? unit / p.kv_heads : 0;
        const int h = in ? (int)(unit - row * p.kv_heads) : 0, b = (int)(row / p.time), t = (int)(row - (long long)b * p.time);
        const long long position = (long long)p.lengths[b] + t;
        const bool live = in && t < (p.counts ? min(p.counts[b], p.time) : p.time) && position >= 0 && position < p.capacity;
        const bool active = live && sub * 8 < p.dim;
        float f[8] = {};
        if (active) load_values((key ? (const T*)p.k_in + row * p.k_pitch : (const T*)p.v_in + row * p.v_pitch) + h * p.dim + 8 * sub, f);
        const long long at = ((long long)b * p.kv_heads + h) * p.capacity + position;
        if constexpr (INT8) {
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) most = max_or_nan(most, fabsf(f[i]));
            for (int o = 1; o < lanes; o <<= 1) most = max_or_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float scale = __fdiv_rn(most, 127.f);
            int q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = scale > 0.f ? min(max(__float2int_rn(__fdiv_rn(f[i], scale)), -127), 127) : 0;
            if (active) {
                *reinterpret_cast<uint2*>((int8_t*)(key ? p.k : p.v) + at * p.dim + 8 * sub) = make_uint2(pack_bytes(q), pack_bytes(q + 4));
                if (sub == 0) (key ? p.k_scale : p.v_scale)[at] = scale;
            }
        } else if (active) {
            store_values((__nv_bfloat16*)(key ? p.k : p.v) + at * p.dim + 8 * sub, f);
        }
    }
}

template <typename T, bool INT8>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const __grid_constant__ CacheParams p) {
    chain_begin();
    const bool key = blockIdx.y == 0;
    const int sub = threadIdx.x & ((1 << p.lane_bits) - 1);
    if (sub * 8 >= p.dim) return;
    const long long stride = (long long)gridDim.x * (kThreads >> p.lane_bits);
    for (long long unit = (long long)blockIdx.x * (kThreads >> p.lane_bits) + (threadIdx.x >> p.lane_bits); unit < p.units; unit += stride) {
        const long long row = unit / p.kv_heads, b = row / p.count, position = p.start + row - b * p.count;
        const int h = (int)(unit - row * p.kv_heads);
        float f[8] = {};
        if (position < p.lengths[b] && position < p.capacity) {
            const long long at = (b * p.kv_heads + h) * p.capacity + position;
            if constexpr (INT8) {
                const uint2 raw = *reinterpret_cast<const uint2*>((const int8_t*)(key ? p.k : p.v) + at * p.dim + 8 * sub);
                const float scale = (key ? p.k_scale : p.v_scale)[at];
                const uint32_t w[2] = {raw.x, raw.y};
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * scale;
            } else {
                load_values((const __nv_bfloat16*)(key ? p.k : p.v) + at * p.dim + 8 * sub, f);
            }
        }
        store_values((T*)(key ? p.k_read : p.v_read) + (row * p.kv_heads + h) * p.dim + 8 * sub, f);
    }
}

CacheParams cache_params(const qmoe_cache_t* c) {
    CacheParams p = {};
    p.k = (void*)c->k; p.v = (void*)c->v; p.k_scale = (float*)c->k_scale; p.v_scale = (float*)c->v_scale;
    p.lengths = (const int*)c->lengths;
    p.capacity = c->capacity; p.batch = (int)c->batch; p.kv_heads = c->kv_heads; p.dim = c->dim;
    while ((8 << p.lane_bits) < c->dim) ++p.lane_bits;
    return p;
}

dim3 cache_grid(const CacheParams& p) {
    const long long blocks = (p.units + (kThreads >> p.lane_bits) - 1) / (kThreads >> p.lane_bits), most = (long long)sm_count() * 8;
    return dim3((unsigned)(blocks < most ? blocks : most), 2);
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
    if (lengths_out == c->lengths) return fail_arg("cache_append: the new lengths need a buffer of their own");
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
    p.units = c->batch * time * c->kv_heads;
    const dim3 grid = cache_grid(p);
    if (c->dtype == QMOE_INT8) {
        if (dtype == QMOE_BF16) chained(cache_append_kernel<__nv_bfloat16, true>, grid, kThreads, 0, stream, p);
        else chained(cache_append_kernel<float, true>, grid, kThreads, 0, stream, p);
    } else {
        if (dtype == QMOE_BF16) chained(cache_append_kernel<__nv_bfloat16, false>, grid, kThreads, 0, stream, p);
        else chained(cache_append_kernel<float, false>, grid, kThreads, 0, stream, p);
    }
    QMOE_LAUNCH_CHECK("cache_append_kernel");
    return 0;
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
    p.units = c->batch * count * c->kv_heads;
    const dim3 grid = cache_grid(p);
    if (c->dtype == QMOE_INT8) {
        if (dtype == QMOE_BF16) chained(cache_read_kernel<__nv_bfloat16, true>, grid, kThreads, 0, stream, p);
        else chained(cache_read_kernel<float, true>, grid, kThreads, 0, stream, p);
    } else {
        if (dtype == QMOE_BF16) chained(cache_read_kernel<__nv_bfloat16, false>, grid, kThreads, 0, stream, p);
        else chained(cache_read_kernel<float, false>, grid, kThreads, 0, stream, p);
    }
    QMOE_LAUNCH_CHECK("cache_read_kernel");
    return 0;
}
