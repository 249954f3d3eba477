// One token a row by temperature, top-k, top-p and min-p from a given uniform number.
//
// A token's weight exp((x - max) / T) is held as a whole number of 2^-31, its mass.  Sums of whole numbers are the same in any order, so the kept
// set and the token do not depend on how the row was cut up, and need no sorted running sum: "the shortest run of the largest
// that holds p of the mass" is a threshold on the tokens' places, a token's place being the 64-bit number (bits of the logit, made to
// grow with it) : (all ones - index), so that of equal logits the one of lower index comes first.  Kept is what has the place
// c or a higher one, for the least c with mass(above c) < p * mass; for top-k the same with counts.
//
// A cluster of up to eight CTAs works on a row, each with a slice of it in shared memory: the logits are read from HBM once.
//   1  the largest logit (its place), over the cluster
//   2  the masses' sum, and the sum of those that min-p lets through.  Where top-p cannot cut into those any more, or nothing cuts, on to 5
//   3  a bound on how far down the kept tokens reach, from the threads' largest logits: where k of those lie in the upper buckets of
//      a histogram by z = (max - x) / T, so do the k largest of all; the same with p of the mass
//   4  a histogram, counts and masses, of what lies above the bound; its crossing bucket is the only one whose members have to be told
//      apart, and goes to a list in the first CTA, which finds the threshold there.  A bucket too full for the list (thousands
//      of equal logits): the threshold by bisection over the places, every step a question to all CTAs
//   5  every CTA's kept mass; the CTA that holds the drawn number's place walks to it by sums over warps, lanes and elements
#include "common.cuh"

#include <cooperative_groups.h>

namespace qmoe {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCtas = 8;
constexpr int kBuckets = 2048, kPerThread = kBuckets / kThreads;
constexpr int kList = 1024;
constexpr float kOne = 2147483648.f;     // 2^31: the mass of the largest logit's token
constexpr float kLastZ = 22.25f;         // exp(-z) 2^31 < 1/2 from z = 22.2 on: no mass
constexpr long long kMaxVocab = 2000000;         // eight slices of at most kBuckets sums of warps (Shared::table)
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

struct Shared {
    u64 places[kMaxCtas], totals[kMaxCtas], passing[kMaxCtas], kept[kMaxCtas];   // of every CTA, in every CTA
    u64 scratch[kWarps];
    u64 answer_count[kMaxCtas], answer_mass[kMaxCtas];       // first CTA: answers to ASK_ABOVE
    u64 ask_place;                       // what the first CTA asks, in every CTA
    int ask, ask_bucket;
    int bound;                           // the last bucket that counts
    unsigned listed;
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
        u64 table[kBuckets];             // step 5: sums of warps
    };
    uint32_t count[kBuckets];            // first CTA: the cluster's, then of the buckets before
    u64 mass[kBuckets];
    u64 list_place[kList];
    uint32_t list_mass[kList];
    u64 least, selected;
};

__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_at(u64 place) {
    const uint32_t b = (uint32_t)(place >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ u64 place_of(float x, int i) { return (u64)ordered(x) << 32 | (0xffffffffu - (uint32_t)i); }
// (x - largest) / T, in (-infinity, 0]; -infinity for a logit that is none
__device__ __forceinline__ float exponent_of(float x, float largest, float inverse) {
    const float apart = x - largest;
    return x == largest ? 0.f : apart == -INFINITY ? -INFINITY : apart * inverse;
}
__device__ __forceinline__ uint32_t mass_of(float weight) { return __float2uint_rn(weight * kOne); }
__device__ __forceinline__ int bucket_of(float exponent) { return min(kBuckets - 1, (int)(exponent * (-kBuckets / kLastZ))); }

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// over the block, in every thread
__device__ u64 block_sum(u64 v, u64* scratch) {
    v = warp_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = threadIdx.x % 32 < kWarps ? scratch[threadIdx.x % 32] : 0;
    return warp_sum64(v);
}
__device__ u64 block_max(u64 v, u64* scratch) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = threadIdx.x % 32 < kWarps ? scratch[threadIdx.x % 32] : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// sum over the threads before this one
__device__ u64 block_before(u64 v, u64* scratch) {
    u64 upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 other = __shfl_up_sync(0xffffffffu, upto, o);
        if ((int)(threadIdx.x & 31) >= o) upto += other;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 31) scratch[threadIdx.x >> 5] = upto;
    __syncthreads();
    u64 before = upto - v;
    for (int w = 0; w < (int)(threadIdx.x >> 5); ++w) before += scratch[w];
    return before;
}

template <typename T, bool HELD>
__global__ void __launch_bounds__(kThreads)
sample_kernel(const __grid_constant__ SampleParams p) {
    chain_begin();
    constexpr int N = Vec16<T>::N;
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    uint4* held = reinterpret_cast<uint4*>(smem + (sizeof(Shared) + 15) / 16 * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = blockIdx.x / ctas;
    cluster.barrier_arrive();            // waited for ahead of the first store to another CTA: by then all of them run
    // the row in pieces of 16 bytes from the 16-byte boundary at or before its start: element i of piece v is token N v + i - lead
    const T* const x = (const T*)p.logits + row * p.vocab;
    const int lead = (int)(((uintptr_t)x & 15u) / sizeof(T));
    const int first_piece = rank * (p.slice / N), pieces = p.slice / N;
    auto fetch = [&](int v, float* f) {
        const int at = (first_piece + v) * N - lead;
        if (at >= 0 && at + N <= p.vocab) {
            Vec16<T>::unpack(*reinterpret_cast<const uint4*>(x + at), f);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = at + i >= 0 && at + i < p.vocab ? Act<T>::load(x + at + i) : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = isnan(f[i]) ? -INFINITY : f[i] + 0.f;      // + 0: one zero
    };
    auto piece = [&](int v, float* f) {
        if constexpr (HELD) Vec16<T>::unpack(held[v], f);
        else fetch(v, f);
    };
    auto add = [&](int b, uint32_t mass) {
        atomicAdd(&s.own.count[b], 1u);
        if constexpr (HELD) {
            atomicAdd(&s.own.low[b], mass & 0xffffu);
            atomicAdd(&s.own.high[b], mass >> 16);
        } else {
            atomicAdd(&s.own.mass[b], (u64)mass);
        }
    };
    auto token_of = [&](int v, int i) { return (first_piece + v) * N + i - lead; };

    const float temperature = p.temperatures ? p.temperatures[row] : p.temperature;
    const float top_p = p.top_ps ? p.top_ps[row] : p.top_p, min_p = fminf(p.min_ps ? p.min_ps[row] : p.min_p, 1.f);
    const bool greedy = !(temperature > 0.f);
    const float inverse = greedy ? 1.f : __fdiv_rn(1.f, temperature);
    const int top_k = greedy ? 1 : p.top_ks ? p.top_ks[row] : p.top_k;

    // 1
    float most = -INFINITY;
    int most_at = 0;
    for (int v = threadIdx.x; v < pieces; v += kThreads) {
        float f[N];
        fetch(v, f);
        if constexpr (HELD) held[v] = Vec16<T>::pack(f);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (f[i] > most) { most = f[i]; most_at = token_of(v, i); }
    }
    u64 place = block_max(place_of(most, most_at), s.scratch);
    cluster.barrier_wait();
    if (threadIdx.x < ctas) cluster.map_shared_rank(&s, threadIdx.x)->places[rank] = place;
    for (int b = threadIdx.x; b < kBuckets; b += kThreads) s.own.count[b] = s.own.low[b] = s.own.high[b] = 0;
    if (threadIdx.x == 0) s.listed = 0;
    cluster.sync();
    for (int c = 0; c < ctas; ++c) place = max(place, s.places[c]);
    const float largest = logit_at(place);
    if (largest == -INFINITY) {
        if (rank == 0 && threadIdx.x == 0) { p.tokens[row] = -1; p.log_probs[row] = -INFINITY; }
        cluster.sync();
        return;
    }
    // 2
    u64 total = 0, passing = 0;
    for (int v = threadIdx.x; v < pieces; v += kThreads) {
        float f[N];
        piece(v, f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float weight = expf(exponent_of(f[i], largest, inverse));
            const uint32_t mass = mass_of(weight);
            total += mass;
            if (!(weight < min_p)) passing += mass;
        }
    }
    const bool one = top_k == 1, by_count = top_k > 1 && top_k < p.vocab, by_mass = !one && !(top_p >= 1.f);
    if (by_count || by_mass) {
        const float exponent = exponent_of(most, largest, inverse);
        const uint32_t mass = mass_of(expf(exponent));
        if (mass) {
            const int b = bucket_of(exponent);
            add(b, mass);
        }
    }
    total = block_sum(total, s.scratch);
    passing = block_sum(passing, s.scratch);
    if (threadIdx.x < ctas) {
        Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
        other->totals[rank] = total;
        other->passing[rank] = passing;
    }
    cluster.sync();
    total = passing = 0;
    for (int c = 0; c < ctas; ++c) { total += s.totals[c]; passing += s.passing[c]; }

    u64 first = one ? place : 0;         // the least place that is kept
    // top-p cuts into what min-p lets through only if that holds more than p of the mass
    const bool cut = by_count || (by_mass && !((double)passing <= (double)top_p * (double)total));
    if (cut) {
        Shared* lead_cta = cluster.map_shared_rank(&s, 0);
        // the cluster's histogram, an eighth of it by every CTA, and in the first CTA the sums of the buckets before
        auto merge = [&]() {
            const int share = kBuckets / ctas;
            for (int b = rank * share + threadIdx.x; b < (rank + 1) * share; b += kThreads) {
                uint32_t count = 0;
                u64 mass = 0;
                for (int c = 0; c < ctas; ++c) {
                    const Shared* other = cluster.map_shared_rank(&s, c);
                    count += other->own.count[b];
                    if constexpr (HELD) mass += (u64)other->own.low[b] + ((u64)other->own.high[b] << 16);
                    else mass += other->own.mass[b];
                }
                lead_cta->count[b] = count;
                lead_cta->mass[b] = mass;
            }
            cluster.sync();
            if (rank == 0) {
                u64 counts = 0, masses = 0;
                for (int i = 0; i < kPerThread; ++i) { counts += s.count[threadIdx.x * kPerThread + i]; masses += s.mass[threadIdx.x * kPerThread + i]; }
                counts = block_before(counts, s.scratch);
                masses = block_before(masses, s.scratch);
                for (int i = 0; i < kPerThread; ++i) {
                    const int b = threadIdx.x * kPerThread + i;
                    const uint32_t count = s.count[b];
                    const u64 mass = s.mass[b];
                    s.count[b] = (uint32_t)counts;
                    s.mass[b] = masses;
                    counts += count;
                    masses += mass;
                }
                __syncthreads();
            }
        };
        merge();
        // 3
        if (rank == 0) {
            if (threadIdx.x == 0) s.bound = kBuckets - 1;
            __syncthreads();
            for (int b = threadIdx.x; b < kBuckets - 1; b += kThreads)
                if (by_count ? s.count[b + 1] >= (uint32_t)top_k : (double)s.mass[b + 1] >= (double)top_p * (double)total) atomicMin(&s.bound, b);
            __syncthreads();
            if (threadIdx.x < ctas) cluster.map_shared_rank(&s, threadIdx.x)->bound = s.bound;
        }
        cluster.sync();
        const int bound = s.bound;
        for (int b = threadIdx.x; b < kBuckets; b += kThreads) s.own.count[b] = s.own.low[b] = s.own.high[b] = 0;
        __syncthreads();
        // 4
        for (int v = threadIdx.x; v < pieces; v += kThreads) {
            float f[N];
            piece(v, f);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float exponent = exponent_of(f[i], largest, inverse);
                if (!(exponent > -kLastZ)) continue;
                const int b = bucket_of(exponent);
                if (b > bound) continue;
                const uint32_t mass = mass_of(expf(exponent));
                if (!mass) continue;
                add(b, mass);
            }
        }
        cluster.sync();
        merge();
        // The first CTA leads: it asks for a bucket's members, or what lies above a place, until it knows the threshold.
        auto ask = [&](int what, int bucket, u64 at) {          // by the first CTA; every CTA then answers in `answer`
            if (threadIdx.x == 0) s.listed = 0;
            if (threadIdx.x < ctas) {
                Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
                other->ask = what;
                other->ask_bucket = bucket;
                other->ask_place = at;
            }
        };
        auto answer = [&]() {
            cluster.sync();
            const int what = s.ask, bucket = s.ask_bucket;
            const u64 at = s.ask_place;
            if (what == ASK_DONE) return false;
            u64 count = 0, mass = 0;
            for (int v = threadIdx.x; v < pieces; v += kThreads) {
                float f[N];
                piece(v, f);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float exponent = exponent_of(f[i], largest, inverse);
                    if (!(exponent > -kLastZ)) continue;
                    if (what == ASK_LIST) {
                        if (bucket_of(exponent) != bucket) continue;
                        const uint32_t m = mass_of(expf(exponent));
                        if (!m) continue;
                        const unsigned to = atomicAdd(&lead_cta->listed, 1u);
                        if (to < kList) {
                            lead_cta->list_place[to] = place_of(f[i], token_of(v, i));
                            lead_cta->list_mass[to] = m;
                        }
                    } else if (place_of(f[i], token_of(v, i)) > at) {
                        const uint32_t m = mass_of(expf(exponent));
                        count += m != 0;
                        mass += m;
                    }
                }
            }
            if (what == ASK_ABOVE) {
                count = block_sum(count, s.scratch);
                mass = block_sum(mass, s.scratch);
                if (threadIdx.x == 0) { lead_cta->answer_count[rank] = count; lead_cta->answer_mass[rank] = mass; }
            }
            cluster.sync();
            return true;
        };
        if (rank == 0) {
            u64 whole = total;           // of what top-k keeps
            int listed_bucket = -1;
            // kept by count: the number before is below `limit`; by mass: the mass before is 0 or below `threshold`
            auto threshold_of = [&](bool counts, u64 limit, double threshold) {
                auto keeps = [&](u64 before) { return counts ? before < limit : before == 0 || (double)before < threshold; };
                // the last bucket whose first member is kept
                if (threadIdx.x == 0) s.bound = 0;
                __syncthreads();
                for (int b = threadIdx.x; b < kBuckets; b += kThreads) {
                    const u64 before = counts ? (u64)s.count[b] : s.mass[b];
                    const bool empty = b + 1 < kBuckets ? s.count[b + 1] == s.count[b] : false;
                    if (!empty && keeps(before)) atomicMax(&s.bound, b);
                }
                __syncthreads();
                const int bucket = s.bound;
                __syncthreads();
                if (bucket != listed_bucket) {
                    ask(ASK_LIST, bucket, 0);
                    answer();
                    listed_bucket = bucket;
                }
                const unsigned n = s.listed;
                if (n > kList) {         // too many to compare with one another
                    u64 c = 0, above = 0;
                    for (int bit = 63; bit >= 0; --bit) {
                        ask(ASK_ABOVE, 0, c | ((1ull << bit) - 1));
                        answer();
                        u64 count = 0, mass = 0;
                        for (int r = 0; r < ctas; ++r) { count += s.answer_count[r]; mass += s.answer_mass[r]; }
                        if (!keeps(counts ? count : mass)) c |= 1ull << bit;
                        else above = mass;
                    }
                    listed_bucket = -1;
                    if (counts && c) {   // the mass that is kept: of the places from c on
                        ask(ASK_ABOVE, 0, c - 1);
                        answer();
                        above = 0;
                        for (int r = 0; r < ctas; ++r) above += s.answer_mass[r];
                        whole = above;
                    }
                    return c;
                }
                if (threadIdx.x == 0) { s.least = ~0ull; s.selected = 0; }
                __syncthreads();
                const u64 count_before = s.count[bucket], mass_before = s.mass[bucket];
                for (unsigned i = threadIdx.x; i < n; i += kThreads) {
                    const u64 mine = s.list_place[i];
                    u64 before = counts ? count_before : mass_before;
                    for (unsigned j = 0; j < n; ++j)
                        if (s.list_place[j] > mine) before += counts ? 1u : s.list_mass[j];
                    if (keeps(before)) {
                        atomicMin(&s.least, mine);
                        atomicAdd(&s.selected, (u64)s.list_mass[i]);
                    }
                }
                __syncthreads();
                if (counts) whole = mass_before + s.selected;
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
    auto kept_of = [&](float f, int v, int i) -> uint32_t {
        const float exponent = exponent_of(f, largest, inverse);
        if (!(exponent > -kLastZ) || place_of(f, token_of(v, i)) < first) return 0u;
        const float weight = expf(exponent);
        return weight < min_p ? 0u : mass_of(weight);
    };
    u64 sum = 0, before = 0, all = 0;
    if (first) {
        for (int v = threadIdx.x; v < pieces; v += kThreads) {
            float f[N];
            piece(v, f);
#pragma unroll
            for (int i = 0; i < N; ++i) sum += kept_of(f[i], v, i);
        }
        sum = block_sum(sum, s.scratch);
        if (threadIdx.x < ctas) cluster.map_shared_rank(&s, threadIdx.x)->kept[rank] = sum;
        cluster.sync();
    }
    for (int c = 0; c < ctas; ++c) {
        const u64 share = first ? s.kept[c] : s.passing[c];
        if (c == rank) { before = all; sum = share; }
        all += share;
    }
    long long drawn = (long long)((double)p.uniforms[row] * (double)all);
    drawn = max(0ll, min(drawn, (long long)all - 1));
    const u64 target = (u64)drawn;
    if (target >= before && target < before + sum) {         // the same for the whole CTA
        const int rounds = (pieces + kThreads - 1) / kThreads;
        for (int r = 0; r < rounds; ++r) {
            const int v = r * kThreads + threadIdx.x;
            u64 mine = 0;
            if (v < pieces) {
                float f[N];
                piece(v, f);
#pragma unroll
                for (int i = 0; i < N; ++i) mine += kept_of(f[i], v, i);
            }
            mine = warp_sum64(mine);
            if (lane == 0) s.table[r * kWarps + warp] = mine;
        }
        __syncthreads();
        if (warp == 0) {
            // the warp's share of the table: 32 sums at a time
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
                const int entry = at + which, v = entry / kWarps * kThreads + entry % kWarps * 32 + lane;
                float f[N];
                uint32_t masses[N];
                u64 lane_sum = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) masses[i] = 0;
                if (v < pieces) {
                    piece(v, f);
#pragma unroll
                    for (int i = 0; i < N; ++i) lane_sum += masses[i] = kept_of(f[i], v, i);
                }
                u64 lane_upto = lane_sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 other = __shfl_up_sync(0xffffffffu, lane_upto, o);
                    if (lane >= o) lane_upto += other;
                }
                u64 running = before + lane_upto - lane_sum;
                if (target >= running && target < running + lane_sum) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        if (target >= running && target < running + masses[i]) {
                            p.tokens[row] = token_of(v, i);
                            p.log_probs[row] = (float)((double)exponent_of(f[i], largest, inverse) - log((double)total / (double)kOne));
                        }
                        running += masses[i];
                    }
                }
                break;
            }
        }
    }
    cluster.sync();                      // nobody leaves while its shared memory is being read
}

template <typename T, bool HELD>
int launch(const SampleParams& p, int ctas, long long rows, cudaStream_t stream) {
    const size_t shared = (sizeof(Shared) + 15) / 16 * 16 + (HELD ? (size_t)p.slice * sizeof(T) : 0);
    QMOE_CUDA(cudaFuncSetAttribute(sample_kernel<T, HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared));
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
    (void)cudaLaunchKernelEx(&config, sample_kernel<T, HELD>, p);
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
    // As many CTAs to a row as have 2048 tokens each, and for few rows up to eight, so that the slices' 32 KB leave room for two CTAs on an SM
    const int size = a->dtype == QMOE_BF16 ? 2 : 4;
    const long long padded = a->vocab + 15;          // a row may start anywhere in its first 16 bytes
    int ctas = 1;
    while (ctas < kMaxCtas && padded > 2048ll * ctas && (a->rows * ctas < 2 * sm_count() || padded * size > 40 * 1024ll * ctas)) ctas *= 2;
    p.slice = (int)((padded + 16 * ctas - 1) / (16 * ctas) * 16);
    const bool held = (long long)p.slice * size <= kMaxSlice && p.slice <= kMaxHeld;
    if (a->dtype == QMOE_BF16) return held ? launch<__nv_bfloat16, true>(p, ctas, a->rows, stream) : launch<__nv_bfloat16, false>(p, ctas, a->rows, stream);
    return held ? launch<float, true>(p, ctas, a->rows, stream) : launch<float, false>(p, ctas, a->rows, stream);
}
