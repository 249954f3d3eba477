// Attention of new queries over a prefix of keys and values that all sequences of a batch share and over each sequence's own cache:
//     out = softmax([q Kp^T, q Kb^T] / sqrt(dim)) [Vp; Vb],
// the prefix read once for the whole batch.  A softmax over a set of keys is joined from its parts: a part that has seen the keys S leaves
// m = max s, l = sum exp(s - m), o = sum exp(s - m) v, and parts meet as M = max m, sum exp(m - M) o / sum exp(m - M) l.
//
// Work items.  All queries that meet the same keys are rows of one product: for the prefix the batch * time * group queries of a
// key/value head, for a sequence's own cache its time * group.  An item is one key/value head, a tile of rows, and a chunk of the
// keys; a chunk of several is joined with the others of its row by prefix_join_kernel.
#include "common.cuh"
#include "tc_ptx.cuh"

namespace qmoe {

int cache_check(const qmoe_cache_t* c);

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kKeys = 64;                // keys of a tile
constexpr int kStages = 3;
constexpr float kLog2e = 1.4426950408889634f;

struct Keys {                            // the prefix, or the sequences' caches
    const uint8_t* k;
    const uint8_t* v;
    const float* k_scale;
    const float* v_scale;
    const int* lengths;
    long long capacity;
    int longest;                         // the host's bound on the lengths
    int row_tiles, splits, chunk;        // tiles of rows per key/value head (and sequence), chunks of keys, keys of a chunk
    int first_slot;                      // of its chunks among a row's parts
};

struct PrefixParams {
    Keys prefix, own;
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    float* lse;
    float2* part_ml;                     // [slots][rows]: m in raw scores, l
    float* part_o;                       // [slots][rows][dim]
    long long rows;                      // batch * time * heads
    int batch, time, kv_heads, group, slots;
    int prefix_items;
    float scale;                         // 1 / sqrt(dim)
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
// two numbers as bf16, and what that leaves of them
__device__ __forceinline__ void split2(float a, float b, uint32_t& high, uint32_t& rest) {
    high = pack2(a, b);
    rest = pack2(a - __uint_as_float(high << 16), b - __uint_as_float(high & 0xffff0000u));
}
// 16 bytes into shared memory, zeros where there is nothing to read
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t at, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t at, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t load_shared(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float2 load_shared_f2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
// D += A B, A 16 x 16 (rows g and g + 8 of lane 4 g + t), B 16 x 8, fp32
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two signed bytes, in the low halves of `w`, as bf16: the low seven bits behind the exponent of 128 give 128 + low, the sign bit
// there gives 128 or 256, and the difference of the two is the byte, exactly.
__device__ __forceinline__ uint32_t bytes_to_bf16(uint32_t w) {
    const uint32_t low = (w & 0x007f007fu) | 0x43004300u, sign = (w & 0x00800080u) | 0x43004300u;
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(low), "r"(sign));
    return r;
}

template <int DIM, bool INT8> struct Tile {
    static constexpr int kRowBytes = INT8 ? DIM : 2 * DIM;
    static constexpr int kPitch = kRowBytes + 16;                  // 16 more: no two of the rows read together share a bank
    static constexpr int kBytes = kKeys * kPitch;
    static constexpr int kStage = 2 * kBytes + (INT8 ? 2 * kKeys * 4 : 0);
    static constexpr int kJoin = kWarps * 16 * (DIM + 4) * 4;      // the warps' parts, where they share the keys
    static constexpr int kShared = kStages * kStage > kJoin ? kStages * kStage : kJoin;
};

// Rows of a tile: 16 to a warp (BY_KEYS false: 64 rows, every warp walks all keys) or the same 16 for all warps (BY_KEYS: a
// quarter of every tile of keys each, joined at the end), for the few rows of one sequence.
template <int DIM, bool INT8, bool BY_KEYS>
__device__ __forceinline__ void attend(const PrefixParams& p, const Keys& keys, uint8_t* smem, int b, int g, int row_tile, int split, bool own) {
    using L = Tile<DIM, INT8>;
    constexpr int ROWS = BY_KEYS ? 16 : 16 * kWarps, NT = BY_KEYS ? kKeys / 8 / kWarps : kKeys / 8, COLS = DIM / 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, t4 = lane & 3;
    const int rows = own ? p.time * p.group : p.batch * p.time * p.group, row0 = row_tile * ROWS + (BY_KEYS ? 0 : 16 * warp);
    const int length = min(max(keys.lengths[b], 0), keys.longest);
    const int begin = split * keys.chunk, end = min(length, begin + keys.chunk);
    // this lane's two rows: where they lie among all rows, and how many keys they see
    long long at[2];
    int limit[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int m = row0 + quad + 8 * i, step = m / p.group;
        const bool in = m < rows;
        at[i] = in ? (((own ? (long long)b * p.time : 0) + step) * p.kv_heads + g) * p.group + (m - step * p.group) : -1;
        limit[i] = !in ? 0 : own ? min(end, length - p.time + step + 1) : end;
    }
    uint32_t qf[DIM / 16][4];
#pragma unroll
    for (int kk = 0; kk < DIM / 16; ++kk)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // a lane's four elements of 16: two and two eight apart as the instruction numbers them; for 8-bit keys they are four
            // neighbours instead (one word of the key), the same permutation of the contraction on both sides
            const __nv_bfloat16* src = p.q + (at[i] < 0 ? 0 : at[i]) * DIM + kk * 16;
            uint2 v;
            if (INT8) v = *reinterpret_cast<const uint2*>(src + 4 * t4);
            else v = make_uint2(*reinterpret_cast<const uint32_t*>(src + 2 * t4), *reinterpret_cast<const uint32_t*>(src + 2 * t4 + 8));
            qf[kk][i] = at[i] < 0 ? 0u : v.x;
            qf[kk][2 + i] = at[i] < 0 ? 0u : v.y;
        }

    const uint32_t base = smem_u32(smem);
    const long long head = ((own ? (long long)b * p.kv_heads : 0) + g) * keys.capacity;
    auto fetch = [&](int tile) {         // keys begin + 64 tile ..; behind `end` zeros, whatever lies there
        const uint32_t stage = base + (tile % kStages) * L::kStage;
        const int first = begin + tile * kKeys;
        constexpr int PIECES = L::kRowBytes / 16;
#pragma unroll
        for (int i = threadIdx.x; i < kKeys * PIECES; i += kThreads) {
            const int key = i / PIECES, piece = i % PIECES;
            const bool there = first + key < end;
            const long long from = (head + (there ? first + key : 0)) * L::kRowBytes + piece * 16;
            copy16(stage + key * L::kPitch + piece * 16, keys.k + from, there);
            copy16(stage + L::kBytes + key * L::kPitch + piece * 16, keys.v + from, there);
        }
        if (INT8) {
            const int key = threadIdx.x & (kKeys - 1);
            const bool there = first + key < end, value = threadIdx.x >= kKeys;
            copy4(stage + 2 * L::kBytes + threadIdx.x * 4, (value ? keys.v_scale : keys.k_scale) + head + (there ? first + key : 0), there);
        }
    };

    float o[COLS][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < COLS; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
    const int tiles = end > begin ? (end - begin + kKeys - 1) / kKeys : 0;
    const float scale2 = p.scale * kLog2e;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        if (s < tiles) fetch(s);
        copies_commit();
    }
    for (int j = 0; j < tiles; ++j) {
        copies_wait<kStages - 2>();
        __syncthreads();                 // tile j is here, and nobody reads the stage that is filled next
        if (j + kStages - 1 < tiles) fetch(j + kStages - 1);
        copies_commit();
        const uint32_t k_tile = base + (j % kStages) * L::kStage, v_tile = k_tile + L::kBytes, scales = k_tile + 2 * L::kBytes;
        const int key0 = BY_KEYS ? warp * 16 : 0, first = begin + j * kKeys + key0;
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
            if constexpr (INT8) {
                const uint32_t row = k_tile + (key0 + 8 * n + quad) * L::kPitch + 4 * t4;
#pragma unroll
                for (int kk = 0; kk < DIM / 16; ++kk) {
                    const uint32_t w = load_shared(row + kk * 16);
                    mma(s[n], qf[kk], bytes_to_bf16(__byte_perm(w, 0, 0x4140)), bytes_to_bf16(__byte_perm(w, 0, 0x4342)));
                }
                const float2 ks = load_shared_f2(scales + (key0 + 8 * n + 2 * t4) * 4);
                s[n][0] *= ks.x; s[n][1] *= ks.y; s[n][2] *= ks.x; s[n][3] *= ks.y;
            } else {
                const uint32_t row = k_tile + (key0 + 8 * n + (lane & 7)) * L::kPitch + (lane >> 3) * 16;
#pragma unroll
                for (int kk = 0; kk < DIM / 16; kk += 2) {
                    uint32_t r[4];
                    ldmatrix4(row + kk * 32, r);
                    mma(s[n], qf[kk], r[0], r[1]);
                    mma(s[n], qf[kk + 1], r[2], r[3]);
                }
            }
        }
        if (first + NT * 8 > min(limit[0], limit[1])) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (first + 8 * n + 2 * t4 + (i & 1) >= limit[i >> 1]) s[n][i] = -INFINITY;
        }
        float alpha[2], base2[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float peak = -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; ++n) peak = fmaxf(peak, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
            const float next = fmaxf(m[i], peak);
            base2[i] = next == -INFINITY ? 0.f : next;        // a row that has seen nothing yet
            alpha[i] = exp2_fast((m[i] - base2[i]) * scale2);
            m[i] = next;
            l[i] *= alpha[i];
        }
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            o[c][0] *= alpha[0]; o[c][1] *= alpha[0];
            o[c][2] *= alpha[1]; o[c][3] *= alpha[1];
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[n][i] = exp2_fast((s[n][i] - base2[i >> 1]) * scale2);
                l[i >> 1] += s[n][i];
            }
            if constexpr (INT8) {        // the value's scale goes with its probability
                const float2 vs = load_shared_f2(scales + (kKeys + key0 + 8 * n + 2 * t4) * 4);
                s[n][0] *= vs.x; s[n][1] *= vs.y; s[n][2] *= vs.x; s[n][3] *= vs.y;
            }
        }
#pragma unroll
        for (int ks = 0; ks < NT / 2; ++ks) {
            // probabilities as two bf16 numbers each, what one leaves in the other: 2^-17 of them is lost, so that the output's own rounding
            // is the only one that shows
            uint32_t a[4], rest[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split2(s[2 * ks + (i >> 1)][2 * (i & 1)], s[2 * ks + (i >> 1)][2 * (i & 1) + 1], a[i], rest[i]);
            if constexpr (INT8) {
                // a word of each of the lane's four keys: columns 32 blk + 4 quad + j of the values, j = 0 .. 3, are the column
                // `quad` of four products
                const uint32_t row = v_tile + (key0 + 16 * ks + 2 * t4) * L::kPitch + 4 * quad;
#pragma unroll
                for (int blk = 0; blk < DIM / 32; ++blk) {
                    const uint32_t w0 = load_shared(row + blk * 32), w1 = load_shared(row + blk * 32 + L::kPitch);
                    const uint32_t w8 = load_shared(row + blk * 32 + 8 * L::kPitch), w9 = load_shared(row + blk * 32 + 9 * L::kPitch);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t b0 = bytes_to_bf16(__byte_perm(w0, w1, 0x0400 + c * 0x101)), b1 = bytes_to_bf16(__byte_perm(w8, w9, 0x0400 + c * 0x101));
                        mma(o[4 * blk + c], a, b0, b1);
                        mma(o[4 * blk + c], rest, b0, b1);
                    }
                }
            } else {
                const uint32_t row = v_tile + (key0 + 16 * ks + (lane & 15)) * L::kPitch + (lane >> 4) * 16;
#pragma unroll
                for (int c = 0; c < COLS; c += 2) {
                    uint32_t r[4];
                    ldmatrix4_trans(row + c * 16, r);
                    mma(o[c], a, r[0], r[1]);
                    mma(o[c + 1], a, r[2], r[3]);
                    mma(o[c], rest, r[0], r[1]);
                    mma(o[c + 1], rest, r[2], r[3]);
                }
            }
        }
    }
    copies_wait<0>();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    // column of element e of product c: see above
    auto column = [&](int c, int e) { return INT8 ? (c >> 2) * 32 + 8 * t4 + 4 * e + (c & 3) : 8 * c + 2 * t4 + e; };
    if constexpr (BY_KEYS) {
        // rows [warp][16][DIM + 4] with m and l behind the row's DIM values
        float* part = reinterpret_cast<float*>(smem);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float* row = part + (warp * 16 + quad + 8 * i) * (DIM + 4);
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                row[column(c, 0)] = o[c][2 * i];
                row[column(c, 1)] = o[c][2 * i + 1];
            }
            if (t4 == 0) { row[DIM] = m[i]; row[DIM + 1] = l[i]; }
        }
        __syncthreads();
        // eight lanes to a row
        const int r = threadIdx.x >> 3, piece = threadIdx.x & 7, mine = row_tile * ROWS + r;
        if (mine >= rows) return;
        const int step = mine / p.group;
        const long long to = (((own ? (long long)b * p.time : 0) + step) * p.kv_heads + g) * p.group + (mine - step * p.group);
        float top = -INFINITY, total = 0.f, factor[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part[(w * 16 + r) * (DIM + 4) + DIM]);
        const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            factor[w] = exp2_fast((part[(w * 16 + r) * (DIM + 4) + DIM] - from) * scale2);
            total += factor[w] * part[(w * 16 + r) * (DIM + 4) + DIM + 1];
        }
        const bool whole = p.slots == 1;
        const long long slot = (long long)(keys.first_slot + split) * p.rows + to;
        const float inverse = total > 0.f ? 1.f / total : 0.f;
        if (piece == 0) {
            if (whole) p.lse[to] = total > 0.f ? top * p.scale + logf(total) : -INFINITY;
            else p.part_ml[slot] = make_float2(top, total);
        }
        for (int d = piece * 4; d < DIM; d += 32) {
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(part + (w * 16 + r) * (DIM + 4) + d);
                sum.x += factor[w] * v.x; sum.y += factor[w] * v.y; sum.z += factor[w] * v.z; sum.w += factor[w] * v.w;
            }
            if (whole) *reinterpret_cast<uint2*>(p.out + to * DIM + d) = make_uint2(pack2(sum.x * inverse, sum.y * inverse), pack2(sum.z * inverse, sum.w * inverse));
            else *reinterpret_cast<float4*>(p.part_o + slot * DIM + d) = sum;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (at[i] < 0) continue;
            const long long slot = (long long)(keys.first_slot + split) * p.rows + at[i];
            const float inverse = l[i] > 0.f ? 1.f / l[i] : 0.f;
            if (t4 == 0) {
                if (p.slots == 1) p.lse[at[i]] = l[i] > 0.f ? m[i] * p.scale + logf(l[i]) : -INFINITY;
                else p.part_ml[slot] = make_float2(m[i], l[i]);
            }
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (p.slots == 1) p.out[at[i] * DIM + column(c, e)] = __float2bfloat16_rn(o[c][2 * i + e] * inverse);
                    else p.part_o[slot * DIM + column(c, e)] = o[c][2 * i + e];
                }
        }
    }
}

template <int DIM, bool INT8, bool PREFIX_BY_KEYS, bool OWN_BY_KEYS>
__global__ void __launch_bounds__(kThreads)
prefix_attention_kernel(const __grid_constant__ PrefixParams p) {
    chain_begin();
    extern __shared__ __align__(16) uint8_t smem[];
    int item = blockIdx.x;
    if (item < p.prefix_items) {
        const int split = item % p.prefix.splits, tile = item / p.prefix.splits;
        attend<DIM, INT8, PREFIX_BY_KEYS>(p, p.prefix, smem, 0, tile % p.kv_heads, tile / p.kv_heads, split, false);
    } else {
        item -= p.prefix_items;
        const int split = item % p.own.splits, tile = item / p.own.splits, head = tile / p.own.row_tiles;
        attend<DIM, INT8, OWN_BY_KEYS>(p, p.own, smem, head / p.kv_heads, head % p.kv_heads, tile % p.own.row_tiles, split, true);
    }
}

// A warp per row: the parts' weights, then their weighted sum
template <int DIM>
__global__ void __launch_bounds__(kThreads)
prefix_join_kernel(const __grid_constant__ PrefixParams p) {
    chain_begin();
    const long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= p.rows) return;
    const float scale2 = p.scale * kLog2e;
    float top = -INFINITY, total = 0.f;
    for (int s = lane; s < p.slots; s += 32) top = fmaxf(top, p.part_ml[s * p.rows + row].x);
    top = warp_max(top);
    const float from = top == -INFINITY ? 0.f : top;
    constexpr int LANES = DIM / 4, TOGETHER = 32 / LANES;        // lanes of a part's row, parts at a time
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = lane / LANES; s < p.slots; s += TOGETHER) {
        const float2 ml = p.part_ml[s * p.rows + row];
        if (ml.y == 0.f) continue;                               // saw no key: its values were not written
        const float factor = exp2_fast((ml.x - from) * scale2);
        const float4 v = *reinterpret_cast<const float4*>(p.part_o + (s * p.rows + row) * DIM + lane % LANES * 4);
        total += factor * ml.y;
        sum.x += factor * v.x; sum.y += factor * v.y; sum.z += factor * v.z; sum.w += factor * v.w;
    }
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
        sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
        sum.z += __shfl_xor_sync(0xffffffffu, sum.z, o);
        sum.w += __shfl_xor_sync(0xffffffffu, sum.w, o);
    }
    const float inverse = total > 0.f ? 1.f / total : 0.f;
    if (lane < LANES) *reinterpret_cast<uint2*>(p.out + row * DIM + lane * 4) = make_uint2(pack2(sum.x * inverse, sum.y * inverse), pack2(sum.z * inverse, sum.w * inverse));
    if (lane == 0) p.lse[row] = total > 0.f ? top * p.scale + logf(total) : -INFINITY;
}

struct Plan { Keys prefix, own; int slots; long long prefix_items, own_items; bool prefix_by_keys, own_by_keys; };

// Chunks of keys: as long as they leave four items to an SM, but not below two tiles.
Plan plan_of(const qmoe_prefix_attention_t* a, const qmoe_cache_t* c) {
    Plan plan = {};
    const long long group = a->heads / c->kv_heads, own_rows = a->time * group, all_rows = c->batch * own_rows;
    plan.prefix_by_keys = all_rows <= 16;
    plan.own_by_keys = own_rows <= 16;
    plan.prefix.row_tiles = ceil_div(all_rows, plan.prefix_by_keys ? 16 : 64);
    plan.own.row_tiles = ceil_div(own_rows, plan.own_by_keys ? 16 : 64);
    const long long prefix_tiles = ceil_div(a->prefix_longest, kKeys), own_tiles = ceil_div(a->longest, kKeys), wanted = (long long)sm_count() * 4;
    const long long prefix_heads = (long long)plan.prefix.row_tiles * c->kv_heads, own_heads = (long long)plan.own.row_tiles * c->kv_heads * c->batch;
    long long chunk = prefix_tiles > own_tiles ? prefix_tiles : own_tiles;
    auto items = [&](long long tiles) { return prefix_heads * ceil_div(prefix_tiles, tiles) + own_heads * ceil_div(own_tiles, tiles); };
    while (chunk > 2 && items(chunk) < wanted) chunk = (chunk + 1) / 2;
    if (chunk < 1) chunk = 1;
    plan.prefix.chunk = plan.own.chunk = (int)chunk * kKeys;
    plan.prefix.splits = ceil_div(prefix_tiles, chunk);
    plan.own.splits = ceil_div(own_tiles, chunk);
    if (!plan.prefix.splits && !plan.own.splits) plan.own.splits = 1;        // nothing to see: zeros are written all the same
    plan.own.first_slot = plan.prefix.splits;
    plan.slots = plan.prefix.splits + plan.own.splits;
    plan.prefix_items = prefix_heads * plan.prefix.splits;
    plan.own_items = own_heads * plan.own.splits;
    return plan;
}

void keys_of(const qmoe_cache_t* c, long long longest, Keys& k) {
    k.k = (const uint8_t*)c->k; k.v = (const uint8_t*)c->v;
    k.k_scale = (const float*)c->k_scale; k.v_scale = (const float*)c->v_scale;
    k.lengths = (const int*)c->lengths; k.capacity = c->capacity; k.longest = (int)longest;
}

int prefix_attention_check(const qmoe_prefix_attention_t* a, const qmoe_cache_t* c, const qmoe_cache_t* prefix) {
    if (!a) return fail_arg("prefix_attention: argument is null");
    if (int rc = cache_check(c)) return rc;
    if (c->dim != 64 && c->dim != 128) return fail_arg("prefix_attention: the head width must be 64 or 128");
    if (a->time <= 0 || a->heads <= 0 || a->heads % c->kv_heads) return fail_arg("prefix_attention: sizes must be positive and heads a multiple of kv_heads");
    if (a->heads > (1 << 20) || a->time > (1ll << 31) / a->heads / c->batch) return fail_arg("prefix_attention: too many rows");
    if (a->longest < 0 || a->longest > c->capacity) return fail_arg("prefix_attention: longest must lie between 0 and the capacity");
    if (prefix) {
        if (int rc = cache_check(prefix)) return rc;
        if (prefix->batch != 1 || prefix->kv_heads != c->kv_heads || prefix->dim != c->dim || prefix->dtype != c->dtype)
            return fail_arg("prefix_attention: the prefix must be a cache of one sequence with the heads, width and dtype of the sequences' cache");
    }
    if (a->prefix_longest < 0 || a->prefix_longest > (prefix ? prefix->capacity : 0)) return fail_arg("prefix_attention: prefix_longest must lie between 0 and the prefix's capacity");
    return 0;
}

template <int DIM, bool INT8>
int launch(const PrefixParams& p, const Plan& plan, cudaStream_t stream) {
    constexpr int SHARED = Tile<DIM, INT8>::kShared;
    auto go = [&](auto kernel) -> int {
        QMOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SHARED));
        chained(kernel, (unsigned)(plan.prefix_items + plan.own_items), kThreads, SHARED, stream, p);
        QMOE_LAUNCH_CHECK("prefix_attention_kernel");
        return 0;
    };
    int rc;
    if (plan.prefix_by_keys) rc = go(prefix_attention_kernel<DIM, INT8, true, true>);        // few rows in all: few in a sequence
    else if (plan.own_by_keys) rc = go(prefix_attention_kernel<DIM, INT8, false, true>);
    else rc = go(prefix_attention_kernel<DIM, INT8, false, false>);
    if (rc || plan.slots == 1) return rc;
    chained(prefix_join_kernel<DIM>, (unsigned)((p.rows + kWarps - 1) / kWarps), kThreads, 0, stream, p);
    QMOE_LAUNCH_CHECK("prefix_join_kernel");
    return 0;
}

}  // namespace
}  // namespace qmoe

using namespace qmoe;

extern "C" int64_t qmoe_prefix_attention_scratch(const qmoe_prefix_attention_t* a, const qmoe_cache_t* c, const qmoe_cache_t* prefix) {
    if (prefix_attention_check(a, c, prefix)) return 0;
    const Plan plan = plan_of(a, c);
    return plan.slots == 1 ? 0 : (int64_t)plan.slots * c->batch * a->time * a->heads * (int64_t)(c->dim + 2) * 4;
}

extern "C" int qmoe_prefix_attention(const qmoe_prefix_attention_t* a, const qmoe_cache_t* c, const qmoe_cache_t* prefix, uint64_t stream_) {
    if (int rc = prefix_attention_check(a, c, prefix)) return rc;
    if (!a->q || !a->out || !a->lse) return fail_arg("prefix_attention: null buffer address");
    if ((a->q | a->out | a->scratch) & 15u || a->lse & 3u) return fail_arg("prefix_attention: buffers must be 16-byte aligned");
    const Plan plan = plan_of(a, c);
    if (plan.slots > 1 && !a->scratch) return fail_arg("prefix_attention: null scratch address");
    if (plan.prefix_items + plan.own_items > 0x7fffffffll) return fail_arg("prefix_attention: too many rows");
    cudaStream_t stream = (cudaStream_t)stream_;
    TimedScope timed(KC_ATTENTION, stream);
    PrefixParams p = {};
    p.prefix = plan.prefix; p.own = plan.own;
    keys_of(prefix ? prefix : c, a->prefix_longest, p.prefix);
    keys_of(c, a->longest, p.own);
    p.q = (const __nv_bfloat16*)a->q; p.out = (__nv_bfloat16*)a->out; p.lse = (float*)a->lse;
    p.rows = c->batch * a->time * a->heads;
    p.part_o = (float*)a->scratch;
    p.part_ml = (float2*)(p.part_o + plan.slots * p.rows * c->dim);
    p.batch = (int)c->batch; p.time = (int)a->time; p.kv_heads = c->kv_heads; p.group = a->heads / c->kv_heads; p.slots = plan.slots;
    p.prefix_items = (int)plan.prefix_items;
    p.scale = 1.f / sqrtf((float)c->dim);
    if (c->dim == 64) return c->dtype == QMOE_INT8 ? launch<64, true>(p, plan, stream) : launch<64, false>(p, plan, stream);
    return c->dtype == QMOE_INT8 ? launch<128, true>(p, plan, stream) : launch<128, false>(p, plan, stream);
}
