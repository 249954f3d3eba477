// What the attention kernels (causal attention, attention over a shared prefix) share: 3-D TMA loads, the pieces of a softmax, bounded
// waits that end a CTA together.
#pragma once
#include "tc_ptx.cuh"

namespace qmoe {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
enum { STATUS_ATTENTION_WAIT = 301 };

__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint32_t dst, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {      // like fmaxf: a number rather than a NaN
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
struct Wait {   // bounded waits of one thread; the first that runs out marks the CTA
    volatile int* abort_flag;
    int* status;
    __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
        if (mbar_wait(bar, parity, abort_flag)) return true;
        if (!*abort_flag) { *abort_flag = 1; atomicExch(status, STATUS_ATTENTION_WAIT); }
        return false;
    }
    // the same for a whole warp: all lanes go on, or none does
    __device__ __forceinline__ bool all(uint32_t bar, uint32_t parity) const { return __all_sync(0xffffffffu, (*this)(bar, parity)); }
};

// a CTA that gave up leaves its copies and MMAs in flight a bounded time to land before its shared memory and TMEM go away
__device__ __forceinline__ void linger_after_abort(const volatile int* abort_flag) {
    if (!*abort_flag) return;
    const unsigned long long start = global_ns();
    while (global_ns() - start < 2000000ull) __nanosleep(1000);
}

}  // namespace
}  // namespace qmoe
