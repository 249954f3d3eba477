// One token a row by temperature, top-k, top-p and min-p from a given uniform number.
//
// A token's weight exp((x - max) / T) is held as a whole number of 2^-31, its mass.  Sums of whole numbers are the same in any order, so the kept
// set and the token do not depend on how the row was cut up, and need no sorted running sum: "the shortest run of the largest
// that holds p of the mass" is a threshold on the tokens' places, a token's place being the 64-bit number (bits of the logit, made to
// grow with it) : (all ones - index), so that of equal logits the one of lower index comes first.  Kept is what has the place
// c or a higher one, for the least c with mass(above c) < p * mass; for top-k the same with counts.
//
// A cluster of up to eight CTAs works on a row, each with a slice of it in shared memory: the logits are read from HBM once.
//   1  the largest logit, over the cluster
//   2  the masses' sum, and the sum of those that min-p lets through.  Where top-p cannot cut into those any more, or nothing cuts, on to 5
//   3  a bound on how far down the kept tokens reach, from the threads' largest logits: where k of those lie in the upper buckets of
//      a histogram by z = (max - x) / T, so do the k largest of all; the same with p of the mass.  What lies above the bound goes to a list in the
//      first CTA; where that holds it (most rows: k or a little more), everything else is done there, each member compared with all others
//   4  else a histogram, counts and masses, of what lies above the bound; its crossing bucket is the only one whose members have to be
//      told apart, and goes to the list instead.  A bucket too full for that (thousands of equal logits): the threshold by bisection over
//      the places, every step a question to all CTAs
//   5  every CTA's kept mass; the warp's share that holds the drawn number's place, by the warps' sums, is looked through by sums over warps, lanes and
//      elements
//
// What bounds it: instructions and the exponential unit (an exponential and a conversion for every token), and for few rows the cluster's barriers.  256 rows
// of 131071 bfloat16 logits by top-p and min-p: 58 us, 67 MB at 1.2 TB/s, 64 % of the issue slots of the SMs that have work; one row of 32000 by top-k and
// top-p: 9.8 us, some 40 % of it the barriers and the launch.  Where thousands of tokens are kept, the histogram's atomics and the passes after it:
// 512 rows of 131071 by top-p 0.95 445 us, 98 without any cut.
#include "common.cuh"

#include <cooperative_groups.h>

#include <type_traits>

namespace qmoe {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kMaxCtas = 8;
constexpr int kTable = 256;
constexpr float kOne = 2147483648.f;     // 2^31: the mass of the largest logit's token
constexpr float kLastZ = 22.25f;         // exp(-z) 2^31 < 1/2 from z = 22.2 on: no mass
constexpr long long kMaxVocab = 2000000;         // eight slices, of which a warp's share has at most kTable sums
constexpr int kMaxSlice = 160 * 1024;    // bytes of a row's slice in shared memory
constexpr int kMaxHeld = 65536;          // its elements

struct SampleParams {
    const void* logits;
    const float* uniforms;
    const float* temperatures;
    const float* top_ps;
    const float* min_ps;
    const int* top_ks;
    long long* tokens;
    float* log_probs;
    int vocab, top_k, slice;             // slice: elements of a CTA, a multiple of 16
    float temperature, top_p, min_p;
};

enum { ASK_DONE = 0, ASK_LIST = 1, ASK_ABOVE = 2 };

template <int kThreads> struct Shared {
    // 256 threads: four such CTAs with slices of 33 KB on an SM instead of the three that twice the sizes leave (512 rows of 131071 by top-p 549 -> 445 us,
    // by min-p 121 -> 108; by top-k 1000, of which the longer list held all, 229 -> 409)
    static constexpr int kBuckets = 2 * kThreads, kList = 4 * kThreads;
    float tops[kMaxCtas];                // of every CTA, in every CTA
    u64 totals[kMaxCtas], passing[kMaxCtas], kept[kMaxCtas];
    u64 scratch[kThreads / 32];
    u64 answer_count[kMaxCtas], answer_mass[kMaxCtas];       // first CTA: answers to ASK_ABOVE
    u64 ask_place;                       // what the first CTA asks, in every CTA
    int ask, ask_bucket;
    int bound;                           // the last bucket that counts
    unsigned staged;                     // members found in this CTA
    unsigned members[kMaxCtas];          // of the list, from every CTA, in every CTA
    u64 least, selected, all;
    union {
        struct {
            // this CTA's.  Masses in two halves of 16 bits, for which shared memory has an addition of its own, while 65536 of them
            // cannot pass 32 bits; larger slices add 64 bits
            uint32_t count[kBuckets];
            union {
                struct { uint32_t low[kBuckets], high[kBuckets]; };
                u64 mass[kBuckets];
            };
        } own;
        struct {                         // while no histogram is being made: this CTA's members; in the first CTA all of them, and masses of up to kThreads
            u64 list[kList];
            uint32_t list_mass[kThreads];
        };
        u64 table[kTable];               // step 5: sums of warps over one warp's share
    };
    u64 picked[kThreads];                // first CTA: the members of one bucket of a long list
    unsigned pickings;
    int bucket;
    uint32_t count[kBuckets];            // first CTA: the cluster's, of the buckets before
    union {
        u64 mass[kBuckets];
        struct { uint32_t low[kBuckets], high[kBuckets]; };      // the masses' halves while they are added up
        float maxima[kMaxCtas * kThreads];       // first CTA: of every thread
    };
};

__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_at(u64 place) {
    const uint32_t b = (uint32_t)(place >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ u64 place_of(float x, int i) { return (u64)ordered(x + 0.f) << 32 | (0xffffffffu - (uint32_t)i); }     // + 0: one zero
// (x - largest) / T, in (-infinity, 0]; -infinity for a logit that is none, NaN stays.  The product says all of that by itself unless the
// largest logit is infinite or 1 / T is 0 or infinite (`odd`)
__device__ __forceinline__ float exponent_of(float x, float largest, float inverse, bool odd) {
    const float apart = x - largest;
    if (odd) return x == largest ? 0.f : apart == -INFINITY ? -INFINITY : apart * inverse;
    return apart * inverse;
}
__device__ __forceinline__ uint32_t mass_of(float weight) { return __float2uint_rn(weight * kOne); }      // of NaN: 0
template <int kBuckets> __device__ __forceinline__ int bucket_of(float exponent) { return min(kBuckets - 1, (int)(exponent * (-kBuckets / kLastZ))); }
__device__ __forceinline__ float max_of(const uint4& v, float so_far, __nv_bfloat16) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(so_far, fmaxf(__low2float(m), __high2float(m)));
}
__device__ __forceinline__ float max_of(const uint4& v, float so_far, float) {
    return fmaxf(so_far, fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w))));
}

// over the warp, in every lane, in three parts of 24, 24 and 16 bits
__device__ __forceinline__ u64 warp_sum64(u64 v) {
    const uint32_t low = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0xffffffu), mid = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 24) & 0xffffffu),
                   high = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 48));
    return (u64)low + ((u64)mid << 24) + ((u64)high << 48);
}
// over the block, in every thread
template <int kThreads> __device__ u64 block_sum(u64 v, u64* scratch) {
    v = warp_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = threadIdx.x % 32 < kThreads / 32 ? scratch[threadIdx.x % 32] : 0;
    return warp_sum64(v);
}
template <int kThreads> __device__ float block_max(float v, u64* scratch) {
    float* values = reinterpret_cast<float*>(scratch);
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) values[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_max(values[threadIdx.x % (kThreads / 32)]);
}
// sum over the threads before this one
template <typename V> __device__ V block_before(V v, u64* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V other = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += other;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = upto;
    __syncthreads();
    const u64 ahead = lane < warp ? scratch[lane] : 0;
    return upto - v + (V)(sizeof(V) == 4 ? __reduce_add_sync(0xffffffffu, (uint32_t)ahead) : warp_sum64(ahead));
}
// list[0 .. n) in falling order; behind it zeros, up to a power of two.  Pairs at most 32 apart stay within a warp's 64 elements.
template <int kThreads> __device__ void sort_falling(u64* list, unsigned n) {
    unsigned padded = 64;
    while (padded < n) padded *= 2;
    __syncthreads();
    for (unsigned i = n + threadIdx.x; i < padded; i += kThreads) list[i] = 0;
    __syncthreads();
    for (unsigned run = 2; run <= padded; run *= 2)
        for (unsigned apart = run / 2; apart; apart /= 2) {
            for (unsigned t = threadIdx.x; t < padded / 2; t += kThreads) {
                const unsigned i = 2 * t - (t & (apart - 1)), j = i + apart;
                const u64 a = list[i], b = list[j];
                if ((a < b) == ((i & run) == 0)) { list[i] = b; list[j] = a; }
            }
            if (apart > 32 || (apart == 1 && run >= 64)) __syncthreads();
            else __syncwarp();
        }
    __syncthreads();
}

template <typename T, bool HELD, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
sample_kernel(const __grid_constant__ SampleParams p) {
    chain_begin();
    constexpr int N = Vec16<T>::N, kWarps = kThreads / 32;
    using Shared = Shared<kThreads>;
    constexpr int kBuckets = Shared::kBuckets, kList = Shared::kList, kPerThread = kBuckets / kThreads;
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    uint4* held = reinterpret_cast<uint4*>(smem + (sizeof(Shared) + 15) / 16 * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = blockIdx.x / ctas;
    cluster.barrier_arrive();            // waited for ahead of the first store to another CTA: by then all of them run
    // the row in pieces of 16 bytes from the 16-byte boundary at or before its start: element i of piece v is token N v + i - lead.  A
    // thread has the same pieces throughout, a warp a run of them, so that its sums say where in the row they lie
    const T* const x = (const T*)p.logits + row * p.vocab;
    const int lead = (int)(((uintptr_t)x & 15u) / sizeof(T));
    const int first_piece = rank * (p.slice / N), pieces = p.slice / N, share = (pieces + kWarps - 1) / kWarps;
    const int begin = warp * share + lane, end = min(pieces, (warp + 1) * share);
    auto token_of = [&](int v, int i) { return (first_piece + v) * N + i - lead; };
    auto inside = [&](int v) { return token_of(v, 0) >= 0 && token_of(v, N) <= p.vocab; };
    auto gather = [&](int v) {           // a piece at the row's ends, or beyond: -infinity where there is no token
        float f[N];
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = token_of(v, i) >= 0 && token_of(v, i) < p.vocab ? Act<T>::load(x + token_of(v, i)) : -INFINITY;
        return Vec16<T>::pack(f);
    };
    auto raw = [&](int v) -> uint4 {
        if constexpr (HELD) return held[v];
        else return inside(v) ? *reinterpret_cast<const uint4*>(x + token_of(v, 0)) : gather(v);
    };
    // this thread's pieces in order; of those that come from memory the next two are asked for meanwhile
    auto each_piece = [&](auto use) __attribute__((always_inline)) {
        if constexpr (HELD) {
            for (int v = begin; v < end; v += 32) use(v, held[v]);
        } else {
            uint4 next = {}, after = {};
            if (begin < end) next = raw(begin);
            if (begin + 32 < end) after = raw(begin + 32);
            for (int v = begin; v < end; v += 32) {
                const uint4 now = next;
                next = after;
                if (v + 64 < end) after = raw(v + 64);
                use(v, now);
            }
        }
    };
    auto each = [&](auto use) __attribute__((always_inline)) {      // the same by element
        each_piece([&](int v, const uint4& d) __attribute__((always_inline)) {
            float f[N];
            Vec16<T>::unpack(d, f);
#pragma unroll
            for (int i = 0; i < N; ++i) use(f[i], v, i);
        });
    };
    auto add = [&](int b, uint32_t mass, bool counts) {
        if (counts) atomicAdd(&s.own.count[b], 1u);
        if constexpr (HELD) {
            atomicAdd(&s.own.low[b], mass & 0xffffu);
            atomicAdd(&s.own.high[b], mass >> 16);
        } else {
            atomicAdd(&s.own.mass[b], (u64)mass);
        }
    };
    auto own_mass = [&](const Shared* of, int b) -> u64 {
        if constexpr (HELD) return (u64)of->own.low[b] + ((u64)of->own.high[b] << 16);
        else return of->own.mass[b];
    };
    if constexpr (HELD) {
        for (int v = begin; v < end; v += 32) {
            if (inside(v)) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(held + v)), "l"(x + token_of(v, 0)) : "memory");
            else held[v] = gather(v);
        }
    }
    const float temperature = p.temperatures ? p.temperatures[row] : p.temperature;
    const float top_p = p.top_ps ? p.top_ps[row] : p.top_p, given_min = p.min_ps ? p.min_ps[row] : p.min_p;
    const float min_p = given_min > 1.f ? 1.f : given_min;       // NaN stays: no weight is below it
    const bool greedy = !(temperature > 0.f);
    const float inverse = greedy ? 1.f : __fdiv_rn(1.f, temperature);
    const int top_k = greedy ? 1 : p.top_ks ? p.top_ks[row] : p.top_k;
    const bool one = top_k == 1, by_count = top_k > 1 && top_k < p.vocab, by_mass = !one && !(top_p >= 1.f);
    const float uniform = p.uniforms[row];
    if (by_count || by_mass)
        for (int b = threadIdx.x; b < kBuckets; b += kThreads) s.own.count[b] = s.own.low[b] = s.own.high[b] = 0;
    if constexpr (HELD) asm volatile("cp.async.wait_all;" ::: "memory");

    // 1
    Shared* const first_cta = cluster.map_shared_rank(&s, 0);
    float largest = -INFINITY;
    each_piece([&](int, const uint4& d) __attribute__((always_inline)) { largest = max_of(d, largest, T()); });
    cluster.barrier_wait();
    if (by_count || by_mass) first_cta->maxima[rank * kThreads + threadIdx.x] = largest;
    largest = block_max<kThreads>(largest, s.scratch);
    if (threadIdx.x < ctas) cluster.map_shared_rank(&s, threadIdx.x)->tops[rank] = largest;
    cluster.sync();
    for (int c = 0; c < ctas; ++c) largest = fmaxf(largest, s.tops[c]);
    if (largest == -INFINITY) {
        if (rank == 0 && threadIdx.x == 0) { p.tokens[row] = -1; p.log_probs[row] = -INFINITY; }
        return;
    }
    const bool odd = largest == INFINITY || inverse == INFINITY || inverse == 0.f;
    auto exponent = [&](float f) { return exponent_of(f, largest, inverse, odd); };
    // 2
    u64 total = 0, passing = 0;
    auto weigh = [&](auto any_odd, auto any_min) __attribute__((always_inline)) {
        each([&](float f, int, int) __attribute__((always_inline)) {
            const float weight = expf(exponent_of(f, largest, inverse, any_odd.value));
            const uint32_t mass = mass_of(weight);
            total += mass;
            if (any_min.value && !(weight < min_p)) passing += mass;
        });
    };
    // 3: the first CTA; top-k's bound needs no masses' sum and comes along with it
    auto find_bound = [&]() __attribute__((always_inline)) {
        for (int i = threadIdx.x; i < ctas * kThreads; i += kThreads) {
            const float e = exponent(s.maxima[i]);
            if (!(e > -kLastZ)) continue;
            const uint32_t mass = mass_of(expf(e));
            if (!mass) continue;
            if (by_count) atomicAdd(&s.own.count[bucket_of<kBuckets>(e)], 1u);
            else add(bucket_of<kBuckets>(e), mass, true);
        }
        __syncthreads();
        // a thread's buckets: the first that reaches what is wanted, together with all before
        uint32_t count[kPerThread], counts = 0;
        u64 mass[kPerThread], masses = 0;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            counts += count[i] = s.own.count[threadIdx.x * kPerThread + i];
            if (!by_count) masses += mass[i] = own_mass(&s, threadIdx.x * kPerThread + i);
        }
        const uint32_t mine = counts;
        counts = block_before(counts, s.scratch);
        if (!by_count) masses = block_before(masses, s.scratch);
        // no bound: all tokens, if few threads have one with a mass, or no list
        if (threadIdx.x == kThreads - 1) s.bound = counts + mine <= kList / 8 ? kBuckets - 1 : kBuckets;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            counts += count[i];
            if (!by_count) masses += mass[i];
            if (by_count ? counts >= (uint32_t)top_k : (double)masses >= (double)top_p * (double)total) {
                atomicMin(&s.bound, threadIdx.x * kPerThread + i);
                break;
            }
        }
        __syncthreads();
        if (threadIdx.x < ctas) cluster.map_shared_rank(&s, threadIdx.x)->bound = s.bound;
    };
    if (by_count && rank == 0) find_bound();
    using Yes = std::true_type;
    using No = std::false_type;
    if (odd) weigh(Yes(), Yes());
    else if (min_p > 0.f) weigh(No(), Yes());
    else weigh(No(), No());
    total = block_sum<kThreads>(total, s.scratch);
    passing = odd || min_p > 0.f ? block_sum<kThreads>(passing, s.scratch) : total;        // its warps' sums stay for step 5
    if (threadIdx.x < ctas) {
        Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
        other->totals[rank] = total;
        other->passing[rank] = passing;
    }
    cluster.sync();
    total = passing = 0;
    for (int c = 0; c < ctas; ++c) { total += s.totals[c]; passing += s.passing[c]; }
    auto finish = [&](int token, float f) {
        p.tokens[row] = token;
        p.log_probs[row] = (float)((double)exponent(f) - log((double)total / (double)kOne));
    };
    auto target_of = [&](u64 all) -> u64 {
        const long long drawn = (long long)((double)uniform * (double)all);
        return one ? 0 : (u64)max(0ll, min(drawn, (long long)all - 1));
    };

    u64 first = one ? (u64)ordered(largest + 0.f) << 32 : 0;         // the least place that is kept
    // top-p cuts into what min-p lets through only if that holds more than p of the mass
    const bool cut = by_count || (by_mass && !((double)passing <= (double)top_p * (double)total));
    if (cut) {
        // 3, by mass
        if (!by_count) {
            if (rank == 0) find_bound();
            cluster.sync();
        }
        const int bound = s.bound;
        // The members of bucket `only`, or of all up to the bound, to the first CTA's list, if it holds them: to the own one first, from where they
        // follow those of the CTAs before.  Their number, or one beyond the list's size.
        auto enlist = [&](int only) __attribute__((always_inline)) -> unsigned {
            constexpr float kScale = -kBuckets / kLastZ;
            const int last = only < 0 ? bound : only;
            const float from = (float)max(only, 0), to = last + 1 < kBuckets ? (float)(last + 1) : INFINITY;      // bucket_of without its conversion
            __syncthreads();
            if (threadIdx.x == 0) s.staged = 0;
            __syncthreads();
            const bool thin = to > kScale * -20.f;       // weights that may have no mass
            bool full = false;
            each_piece([&](int v, const uint4& d) __attribute__((always_inline)) {
                if (full) return;
                float f[N];
                Vec16<T>::unpack(d, f);
                unsigned members = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float e = exponent(f[i]), at = e * kScale;
                    if (e > -kLastZ && at >= from && at < to) members |= 1u << i;
                }
                if (thin)
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (members >> i & 1 && mass_of(expf(exponent(f[i]))) == 0) members ^= 1u << i;
                if (!members) return;
                unsigned where = atomicAdd(&s.staged, (unsigned)__popc(members));
                full = where + __popc(members) > kList;
                if (full) return;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (members >> i & 1) s.list[where++] = place_of(f[i], token_of(v, i));
            });
            __syncthreads();
            const unsigned mine = s.staged;
            if (threadIdx.x < ctas) cluster.map_shared_rank(&s, threadIdx.x)->members[rank] = mine;
            cluster.sync();
            unsigned n = 0, ahead = 0;
#pragma unroll
            for (int c = 0; c < kMaxCtas; ++c) {
                if (c == rank) ahead = n;
                if (c < ctas) n += s.members[c];
            }
            if (n <= kList && rank)
                for (unsigned i = threadIdx.x; i < mine; i += kThreads) first_cta->list[ahead + i] = s.list[i];
            cluster.sync();
            return n;
        };
        // sums of the buckets before, in place
        auto accumulate = [&]() __attribute__((always_inline)) {
            __syncthreads();
            u64 counts = 0, masses = 0, mass[kPerThread];
            uint32_t count[kPerThread];
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                counts += count[i] = s.count[threadIdx.x * kPerThread + i];
                masses += mass[i] = s.mass[threadIdx.x * kPerThread + i];
            }
            counts = block_before(counts, s.scratch);
            masses = block_before(masses, s.scratch);
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const int b = threadIdx.x * kPerThread + i;
                s.count[b] = (uint32_t)counts;
                s.mass[b] = masses;
                counts += count[i];
                masses += mass[i];
            }
            if (threadIdx.x == kThreads - 1) s.all = masses;
            __syncthreads();
        };
        auto weight_at = [&](u64 at) { return expf(exponent(logit_at(at))); };
        // Of n <= kThreads places in shared memory: kept by count, the number before (and `base` of them ahead of all) below `limit`; by mass, the mass
        // before 0 or below `threshold`.  s.least: the least place that is kept, all ones for none; s.selected: the kept ones' mass.
        // Few are compared with all others, by as many lanes as there are for each, more are sorted (512 rows of 131071 bfloat16 logits, some 200 of them equal ones: 671 and 549 us).
        auto compare = [&](u64* places, unsigned n, bool counts, u64 base, u64 limit, double threshold) __attribute__((always_inline)) {
            u64 at, mass_ahead = 0;
            uint32_t mass;
            unsigned ahead = 0;
            bool leads;
            if (threadIdx.x == 0) { s.least = ~0ull; s.selected = 0; }
            if (n > kThreads / 4) {
                sort_falling<kThreads>(places, n);
                ahead = threadIdx.x;
                leads = ahead < n;
                at = leads ? places[ahead] : 0;
                mass = leads ? mass_of(weight_at(at)) : 0u;
                mass_ahead = block_before((u64)mass, s.scratch);
            } else {
                int bits = 0;
                while (bits < 5 && n << (bits + 1) <= kThreads) ++bits;
                const unsigned me = threadIdx.x >> bits, of = 1u << bits;
                at = me < n ? places[me] : 0;
                mass = me < n ? mass_of(weight_at(at)) : 0u;
                leads = me < n && (threadIdx.x & (of - 1)) == 0;
                if (leads) s.list_mass[me] = mass;
                __syncthreads();
                for (unsigned j = threadIdx.x & (of - 1); j < n; j += of)
                    if (places[j] > at) {
                        ++ahead;
                        mass_ahead += s.list_mass[j];
                    }
                for (unsigned o = 1; o < of; o <<= 1) {
                    ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
                    mass_ahead += __shfl_xor_sync(0xffffffffu, mass_ahead, o);
                }
            }
            // the kept ones are a run from the highest: the last of them, by which no other follows that is kept, is the one to know
            auto keeps = [&](u64 number, u64 mass_before) {
                const u64 before = base + (counts ? number : mass_before);
                return counts ? before < limit : before == 0 || (double)before < threshold;
            };
            if (leads && keeps(ahead, mass_ahead) && (ahead + 1 == n || !keeps(ahead + 1, mass_ahead + mass))) {
                s.least = at;
                s.selected = mass_ahead + mass;
            }
            __syncthreads();
        };
        // the places of the list that `in` takes, to s.picked; their number, which may be more than fit there
        auto pick = [&](unsigned n, auto in) __attribute__((always_inline)) -> unsigned {
            if (threadIdx.x == 0) s.pickings = 0;
            __syncthreads();
            for (unsigned i = threadIdx.x; i < n; i += kThreads) {
                const u64 at = s.list[i];
                if (!in(at)) continue;
                const unsigned to = atomicAdd(&s.pickings, 1u);
                if (to < kThreads) s.picked[to] = at;
            }
            __syncthreads();
            return s.pickings;
        };
        // a histogram of the list over `bucket`, then sums of the buckets before
        auto spread = [&](unsigned n, auto bucket) __attribute__((always_inline)) {
            __syncthreads();             // the one before has been read
            for (int b = threadIdx.x; b < kBuckets; b += kThreads) s.count[b] = s.low[b] = s.high[b] = 0;
            __syncthreads();
            for (unsigned i = threadIdx.x; i < n; i += kThreads) {
                const u64 at = s.list[i];
                const int b = bucket(at);
                if (b < 0) continue;
                const uint32_t mass = mass_of(weight_at(at));
                atomicAdd(&s.count[b], 1u);
                atomicAdd(&s.low[b], mass & 0xffffu);
                atomicAdd(&s.high[b], mass >> 16);
            }
            __syncthreads();
            u64 mass[kPerThread];
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) mass[i] = (u64)s.low[threadIdx.x * kPerThread + i] + ((u64)s.high[threadIdx.x * kPerThread + i] << 16);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) s.mass[threadIdx.x * kPerThread + i] = mass[i];
            accumulate();
        };
        // the last bucket that holds anything and whose sum before `keeps`
        auto crossing = [&](auto keeps) __attribute__((always_inline)) {
            if (threadIdx.x == 0) s.bucket = 0;
            __syncthreads();
            for (int b = threadIdx.x; b < kBuckets; b += kThreads)
                if ((b + 1 == kBuckets || s.mass[b + 1] != s.mass[b]) && keeps(b)) atomicMax(&s.bucket, b);
            __syncthreads();
            const int found = s.bucket;
            __syncthreads();
            return found;
        };
        // Of the first CTA's sorted list: kept by count, the number before (and `base` of them ahead of the list) below `limit`; by mass, the mass
        // before 0 or below `threshold`.  The least place that is kept, all ones for none; `selected` becomes the kept members' mass.
        constexpr int EACH = kList / kThreads;
        auto least_kept = [&](unsigned n, bool counts, u64 base, u64 limit, double threshold) __attribute__((always_inline)) {
            if (threadIdx.x == 0) { s.least = ~0ull; s.selected = 0; }
            u64 mass[EACH], sum = 0;
            const unsigned begin = threadIdx.x * EACH;
#pragma unroll
            for (int i = 0; i < EACH; ++i) sum += mass[i] = begin + i < n ? mass_of(weight_at(s.list[begin + i])) : 0;
            const u64 mass_before = block_before(sum, s.scratch);
            u64 before = mass_before;
            int kept = 0;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const u64 so_far = base + (counts ? begin + i : before);
                if (begin + i < n && (counts ? so_far < limit : so_far == 0 || (double)so_far < threshold)) {
                    before += mass[i];
                    ++kept;
                }
            }
            // what is kept is a run from the front: its last member says where it ends
            if (kept && (kept < EACH || begin + EACH >= n)) { s.least = s.list[begin + kept - 1]; s.selected = before; }
            if (kept == EACH && begin + EACH < n) {
                const u64 so_far = base + (counts ? begin + EACH : before);
                if (!(counts ? so_far < limit : (double)so_far < threshold)) { s.least = s.list[begin + EACH - 1]; s.selected = before; }
            }
            __syncthreads();
        };
        if (bound < kBuckets) {          // everything that can be kept, if the list holds it
            const unsigned n = enlist(-1);
            if (n <= kList) {            // the first CTA alone goes on
                if (rank) return;
                if (n <= kThreads) {     // a short list: every member compared with all others, by as many lanes as there are for each
                    int bits = 0;
                    while (bits < 5 && n << (bits + 1) <= kThreads) ++bits;
                    const unsigned me = threadIdx.x >> bits, of = 1u << bits;
                    const u64 at = me < n ? s.list[me] : 0;
                    const float weight = me < n ? weight_at(at) : 0.f;
                    const uint32_t mass = mass_of(weight);
                    const bool leads = me < n && (threadIdx.x & (of - 1)) == 0;
                    if (leads) s.list_mass[me] = mass;
                    __syncthreads();
                    unsigned ahead = 0;
                    u64 mass_ahead = 0, behind = 0;
                    for (unsigned j = threadIdx.x & (of - 1); j < n; j += of)
                        if (s.list[j] > at) {
                            ++ahead;
                            mass_ahead += s.list_mass[j];
                        }
                    for (unsigned o = 1; o < of; o <<= 1) {
                        ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
                        mass_ahead += __shfl_xor_sync(0xffffffffu, mass_ahead, o);
                    }
                    bool keep = !by_count || ahead < (unsigned)top_k;
                    if (by_mass) {
                        const u64 whole = by_count ? block_sum<kThreads>(leads && keep ? mass : 0u, s.scratch) : total;
                        keep = keep && (mass_ahead == 0 || (double)mass_ahead < (double)top_p * (double)whole);
                    }
                    const uint32_t kept = leads && keep && !(weight < min_p) ? mass : 0u;
                    const u64 target = target_of(block_sum<kThreads>(kept, s.scratch));
                    if (leads) s.list_mass[me] = kept;
                    __syncthreads();
                    for (unsigned j = threadIdx.x & (of - 1); j < n; j += of)      // by index: the places' lower halves fall with it
                        if ((uint32_t)s.list[j] > (uint32_t)at) behind += s.list_mass[j];
                    for (unsigned o = 1; o < of; o <<= 1) behind += __shfl_xor_sync(0xffffffffu, behind, o);
                    if (kept && target >= behind && target < behind + kept) finish((int)(0xffffffffu - (uint32_t)at), logit_at(at));
                    return;
                }
                // A longer one: a finer histogram of it, whose crossing bucket's members are compared; or, should even those be many, sorted
                const float finer = kBuckets * (kBuckets / kLastZ) / (bound + 1);
                auto fine = [&](u64 at) { return min(kBuckets - 1, (int)(exponent(logit_at(at)) * -finer)); };
                u64 whole = total;
                bool spread_out = false;
                auto cut_at = [&](bool counts, u64 limit, double threshold) __attribute__((always_inline)) {
                    if (!spread_out) spread(n, fine);
                    spread_out = true;
                    const int b = crossing([&](int i) {
                        const u64 before = counts ? (u64)s.count[i] : s.mass[i];
                        return counts ? before < limit : before == 0 || (double)before < threshold;
                    });
                    const unsigned members = pick(n, [&](u64 at) { return fine(at) == b; });
                    if (members <= kThreads) {
                        compare(s.picked, members, counts, counts ? (u64)s.count[b] : s.mass[b], limit, threshold);
                        if (counts) whole = s.mass[b] + s.selected;
                    } else {
                        sort_falling<kThreads>(s.list, n);
                        least_kept(n, counts, 0, limit, threshold);
                        if (counts) whole = s.selected;
                    }
                    first = max(first, members ? s.least : 0);          // an empty last bucket: all of them
                    if (counts && !members) whole = total;
                    __syncthreads();
                };
                if (by_count) cut_at(true, (u64)top_k, 0.0);
                if (by_mass) cut_at(false, 0, (double)top_p * (double)whole);
                // the kept ones by index: the bucket of indices in which the drawn number lies, and in it the token
                const unsigned each = (p.vocab + kBuckets - 1) / kBuckets;
                auto index_of = [&](u64 at) { return 0xffffffffu - (uint32_t)at; };
                auto kept_at = [&](u64 at) { return at >= first && !(weight_at(at) < min_p); };
                spread(n, [&](u64 at) { return kept_at(at) ? (int)(index_of(at) / each) : -1; });
                const u64 target = target_of(s.all);
                const int b = crossing([&](int i) { return s.mass[i] <= target; });
                const unsigned members = pick(n, [&](u64 at) { return kept_at(at) && (int)(index_of(at) / each) == b; });
                // (no more than `each` of them: vocabularies beyond 512 * kBuckets tokens may have to look through the list)
                const u64* const among = members <= kThreads ? s.picked : s.list;
                const unsigned many = members <= kThreads ? members : n;
                for (unsigned i = threadIdx.x; i < many; i += kThreads) {
                    const u64 at = among[i];
                    if (!kept_at(at) || (int)(index_of(at) / each) != b) continue;
                    u64 before = s.mass[b];
                    for (unsigned j = 0; j < many; ++j) {
                        const u64 other = among[j];
                        if (index_of(other) < index_of(at) && kept_at(other) && (int)(index_of(other) / each) == b) before += mass_of(weight_at(other));
                    }
                    if (target >= before && target < before + mass_of(weight_at(at))) finish((int)index_of(at), logit_at(at));
                }
                return;
            }
        }
        // 4
        __syncthreads();
        for (int b = threadIdx.x; b < kBuckets; b += kThreads) s.own.count[b] = s.own.low[b] = s.own.high[b] = 0;
        __syncthreads();
        each([&](float f, int, int) __attribute__((always_inline)) {
            const float e = exponent(f);
            if (!(e > -kLastZ)) return;
            const int b = bucket_of<kBuckets>(e);
            if (b > bound) return;
            const uint32_t mass = mass_of(expf(e));
            if (mass) add(b, mass, by_count);         // a bucket with members has mass: only top-k needs their number
        });
        cluster.sync();
        // the cluster's, an equal share of the buckets by every CTA
        for (int b = rank * (kBuckets / ctas) + threadIdx.x; b < (rank + 1) * (kBuckets / ctas); b += kThreads) {
            uint32_t count = 0;
            u64 mass = 0;
#pragma unroll
            for (int c = 0; c < kMaxCtas; ++c)
                if (c < ctas) {
                    const Shared* other = cluster.map_shared_rank(&s, c);
                    count += other->own.count[b];
                    mass += own_mass(other, b);
                }
            first_cta->count[b] = count;
            first_cta->mass[b] = mass;
        }
        cluster.sync();
        // The first CTA leads: it asks for a bucket's members, or what lies above a place, until it knows the threshold.
        auto ask = [&](int what, int bucket, u64 at) __attribute__((always_inline)) {          // by the first CTA; every CTA then answers in `answer`
            if (threadIdx.x < ctas) {
                Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
                other->ask = what;
                other->ask_bucket = bucket;
                other->ask_place = at;
            }
        };
        unsigned listed = 0;
        auto answer = [&]() __attribute__((always_inline)) {
            cluster.sync();
            const int what = s.ask;
            if (what == ASK_DONE) return false;
            if (what == ASK_LIST) {
                listed = enlist(s.ask_bucket);
            } else {
                const u64 at = s.ask_place;
                u64 count = 0, mass = 0;
                each([&](float f, int v, int i) __attribute__((always_inline)) {
                    const float e = exponent(f);
                    if (!(e > -kLastZ) || place_of(f, token_of(v, i)) <= at) return;
                    const uint32_t m = mass_of(expf(e));
                    count += m != 0;
                    mass += m;
                });
                count = block_sum<kThreads>(count, s.scratch);
                mass = block_sum<kThreads>(mass, s.scratch);
                if (threadIdx.x == 0) { first_cta->answer_count[rank] = count; first_cta->answer_mass[rank] = mass; }
                cluster.sync();
            }
            return true;
        };
        if (rank == 0) {
            accumulate();
            u64 whole = total;           // of what top-k keeps
            int listed_bucket = -1;
            auto threshold_of = [&](bool counts, u64 limit, double threshold) __attribute__((always_inline)) -> u64 {
                auto keeps = [&](u64 before) { return counts ? before < limit : before == 0 || (double)before < threshold; };
                const int bucket = crossing([&](int b) { return keeps(counts ? (u64)s.count[b] : s.mass[b]); });      // the last whose first member is kept
                if (bucket != listed_bucket) {
                    ask(ASK_LIST, bucket, 0);
                    answer();
                    listed_bucket = bucket;
                }
                const unsigned n = listed;
                if (n > kList) {         // too many to compare with one another
                    u64 c = 0;
                    for (int bit = 63; bit >= 0; --bit) {
                        ask(ASK_ABOVE, 0, c | ((1ull << bit) - 1));
                        answer();
                        u64 before = 0;
                        for (int r = 0; r < ctas; ++r) before += counts ? s.answer_count[r] : s.answer_mass[r];
                        if (!keeps(before)) c |= 1ull << bit;
                    }
                    listed_bucket = -1;
                    if (counts && c) {   // the mass that is kept: of the places from c on
                        ask(ASK_ABOVE, 0, c - 1);
                        answer();
                        whole = 0;
                        for (int r = 0; r < ctas; ++r) whole += s.answer_mass[r];
                    }
                    return c;
                }
                u64 base = counts ? (u64)s.count[bucket] : s.mass[bucket], mass_base = s.mass[bucket];
                unsigned some = n;
                u64* among = s.list;
                // more than can be compared with one another cheaply: a histogram within the bucket, unless the one at hand is still needed
                if (n > 64 && !(counts && by_mass)) {
                    spread(n, [&](u64 at) {
                        const float within = exponent(logit_at(at)) * (-kBuckets / kLastZ) - bucket;
                        return max(0, min(kBuckets - 1, (int)(within * kBuckets)));
                    });
                    const int b = crossing([&](int i) { return keeps(base + (counts ? (u64)s.count[i] : s.mass[i])); });
                    const unsigned found = pick(n, [&](u64 at) {
                        const float within = exponent(logit_at(at)) * (-kBuckets / kLastZ) - bucket;
                        return max(0, min(kBuckets - 1, (int)(within * kBuckets))) == b;
                    });
                    if (found && found <= kThreads) {
                        base += counts ? (u64)s.count[b] : s.mass[b];
                        mass_base += s.mass[b];
                        among = s.picked;
                        some = found;
                    }
                }
                if (some <= kThreads) {
                    compare(among, some, counts, base, limit, threshold);
                } else {
                    sort_falling<kThreads>(s.list, n);
                    least_kept(n, counts, base, limit, threshold);
                }
                if (counts) whole = mass_base + s.selected;
                const u64 c = n ? s.least : 0;      // an empty last bucket: everything is kept
                __syncthreads();
                return c;
            };
            if (by_count) first = threshold_of(true, (u64)top_k, 0.0);
            if (by_mass) first = max(first, threshold_of(false, 0, (double)top_p * (double)whole));
            ask(ASK_DONE, 0, first);
            answer();
        } else {
            while (answer()) {}
            first = s.ask_place;
        }
    }
    // 5
    const float edge = first ? logit_at(first) : -INFINITY;
    const unsigned edge_token = 0xffffffffu - (uint32_t)first;
    auto kept_of = [&](float f, int v, int i) __attribute__((always_inline)) -> uint32_t {
        const float e = exponent(f);
        if (!(f >= edge) || !(e > -kLastZ) || (f == edge && (unsigned)token_of(v, i) > edge_token)) return 0u;
        const float weight = expf(e);
        return weight < min_p ? 0u : mass_of(weight);
    };
    u64 sum = 0, before = 0, all = 0;
    if (cut || one) {
        each([&](float f, int v, int i) __attribute__((always_inline)) { sum += kept_of(f, v, i); });
        sum = block_sum<kThreads>(sum, s.scratch);
        if (threadIdx.x < ctas) cluster.map_shared_rank(&s, threadIdx.x)->kept[rank] = sum;
        cluster.sync();
    }
    for (int c = 0; c < ctas; ++c) {
        const u64 of_cta = cut || one ? s.kept[c] : s.passing[c];
        if (c == rank) { before = all; sum = of_cta; }
        all += of_cta;
    }
    const u64 target = target_of(all);
    if (target < before || target >= before + sum) return;          // another CTA's
    // the warp in whose share it lies, by the warps' sums; all warps look through that share
    int from, until;
    {
        u64 of_warp = lane < kWarps ? s.scratch[lane] : 0, upto = of_warp;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
        }
        const int which = __ffs(__ballot_sync(0xffffffffu, before + upto > target)) - 1;
        before += __shfl_sync(0xffffffffu, upto - of_warp, which);
        from = which * share;
        until = min(pieces, from + share);
    }
    const int rounds = (until - from + kThreads - 1) / kThreads;
    for (int r = 0; r < rounds; ++r) {
        const int v = from + r * kThreads + threadIdx.x;
        u64 mine = 0;
        if (v < until) {
            float f[N];
            Vec16<T>::unpack(raw(v), f);
#pragma unroll
            for (int i = 0; i < N; ++i) mine += kept_of(f[i], v, i);
        }
        mine = warp_sum64(mine);
        if (lane == 0) s.table[r * kWarps + warp] = mine;
    }
    __syncthreads();
    if (warp) return;
    // 32 sums of the table at a time
    for (int at = 0; at < rounds * kWarps; at += 32) {
        const u64 mine = at + lane < rounds * kWarps ? s.table[at + lane] : 0;
        u64 upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + upto > target);
        if (!hit) {
            before += __shfl_sync(0xffffffffu, upto, 31);
            continue;
        }
        const int which = __ffs(hit) - 1;
        before += __shfl_sync(0xffffffffu, upto - mine, which);
        const int entry = at + which, v = from + entry / kWarps * kThreads + entry % kWarps * 32 + lane;
        float f[N];
        uint32_t masses[N];
        u64 lane_sum = 0;
        if (v < until) Vec16<T>::unpack(raw(v), f);
#pragma unroll
        for (int i = 0; i < N; ++i) lane_sum += masses[i] = v < until ? kept_of(f[i], v, i) : 0u;
        u64 running = lane_sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 other = __shfl_up_sync(0xffffffffu, running, o);
            if (lane >= o) running += other;
        }
        running += before - lane_sum;
        if (target >= running && target < running + lane_sum) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (target >= running && target < running + masses[i]) finish(token_of(v, i), f[i]);
                running += masses[i];
            }
        }
        return;
    }
}

template <typename T, bool HELD, int kThreads>
int launch(const SampleParams& p, int ctas, long long rows, cudaStream_t stream) {
    const size_t shared = (sizeof(Shared<kThreads>) + 15) / 16 * 16 + (HELD ? (size_t)p.slice * sizeof(T) : 0);
    QMOE_CUDA((allow_shared<sample_kernel<T, HELD, kThreads>>((int)shared)));
    cudaLaunchAttribute attributes[2] = {chain_attribute(), {}};
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = ctas;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(rows * ctas));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    config.attrs = attributes;
    config.numAttrs = 2;
    (void)cudaLaunchKernelEx(&config, sample_kernel<T, HELD, kThreads>, p);
    QMOE_LAUNCH_CHECK("sample_kernel");
    return 0;
}

}  // namespace
}  // namespace qmoe

using namespace qmoe;

extern "C" int qmoe_sample(const qmoe_sample_t* a, uint64_t stream_) {
    if (!a) return fail_arg("sample: argument is null");
    if (a->dtype != QMOE_F32 && a->dtype != QMOE_BF16) return fail_arg("sample: dtype must be QMOE_F32 or QMOE_BF16");
    if (a->rows < 0 || a->vocab <= 0 || a->vocab > kMaxVocab || a->rows > (0x7fffffff / kMaxCtas))
        return fail_arg("sample: rows must not be negative, vocab between 1 and %lld", kMaxVocab);
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
    p.vocab = (int)a->vocab; p.top_k = a->top_k; p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p;
    // Few rows: as many CTAs to a row as have 2048 tokens each and find an SM of their own, up to eight, with 512 threads.  Many rows: as
    // few as hold the row in slices of 40 KB, with 256 threads, because what a warp does beside its tokens is half of the work
    const int size = a->dtype == QMOE_BF16 ? 2 : 4;
    const long long padded = a->vocab + 15;          // a row may start anywhere in its first 16 bytes
    int ctas = 1;
    while (ctas < kMaxCtas && padded > 2048ll * ctas && (a->rows * ctas <= sm_count() || padded * size > 40 * 1024ll * ctas)) ctas *= 2;
    p.slice = (int)((padded + 16 * ctas - 1) / (16 * ctas) * 16);
    const bool held = (long long)p.slice * size <= kMaxSlice && p.slice <= kMaxHeld, many = a->rows * ctas > 2 * sm_count();
    if (a->dtype == QMOE_BF16)
        return !held ? launch<__nv_bfloat16, false, 512>(p, ctas, a->rows, stream) : many ? launch<__nv_bfloat16, true, 256>(p, ctas, a->rows, stream)
                                                                                          : launch<__nv_bfloat16, true, 512>(p, ctas, a->rows, stream);
    return !held ? launch<float, false, 512>(p, ctas, a->rows, stream) : many ? launch<float, true, 256>(p, ctas, a->rows, stream)
                                                                              : launch<float, true, 512>(p, ctas, a->rows, stream);
}
