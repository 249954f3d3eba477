// Attention of new queries over a prefix of keys and values that all sequences of a batch share and over each sequence's own cache:
//     out = softmax([q Kp^T, q Kb^T] / sqrt(dim)) [Vp; Vb],
// the prefix read once for the whole batch.  A softmax over a set of keys is joined from its parts: a part that has seen the keys S leaves
// m = max s, l = sum exp(s - m), o = sum exp(s - m) v, and parts meet as M = max m, sum exp(m - M) o / sum exp(m - M) l.
// l = 0 says that a part has seen nothing; a score that is no number leaves m as it is and l NaN, and with it the row.
//
// Work items.  All queries that meet the same keys are rows of one product: for the prefix the batch * time * group queries of a
// key/value head, for a sequence's own cache its time * group.  An item is one key/value head, a tile of rows, and a chunk of the
// keys; a chunk of several is joined with the others of its row by prefix_join_kernel.
#include "common.cuh"
#include "attention_ptx.cuh"

#include <type_traits>

namespace qmoe {

int cache_check(const qmoe_cache_t* c);

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kKeys = 64;                // what chunks of keys are counted in
constexpr float LN2 = 0.6931471805599453f;

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
    float2* part_ml;                     // [slots][rows]: m as an exponent of 2, l
    float* part_o;                       // [slots][rows][dim]
    long long rows;                      // batch * time * heads
    int batch, time, kv_heads, group, slots;
    int prefix_items;
    int checks;                          // some rows do not see all keys of their sequence (see row_again)
    float scale;                         // 1 / sqrt(dim)
};

// Two numbers that are not negative as bf16, cut off and not rounded (the upper halves as they are), and what that leaves of them, rounded: 2^-16
// of a number is lost at most.
__device__ __forceinline__ void split2(float a, float b, uint32_t& high, uint32_t& rest) {
    high = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    float a_rest, b_rest;
    unpair2(add2(pair2(a, b), pair2(__uint_as_float((__float_as_uint(a) & 0xffff0000u) | 0x80000000u),
                                    __uint_as_float((__float_as_uint(b) & 0xffff0000u) | 0x80000000u))), a_rest, b_rest);
    rest = pack2(a_rest, b_rest);
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

// Keys of a tile: 128 where a warp has a quarter of them, so that its steps have some work to overlap: a tile of 64 took 1450 cycles (128 sequences, 8
// heads, up to 1025 positions), in which nothing was waited for but one step for the next
template <int DIM, bool INT8, bool BY_KEYS> struct Tile {
    static constexpr int kKeys = BY_KEYS && DIM == 64 ? 128 : 64;
    static constexpr int kRowBytes = INT8 ? DIM : 2 * DIM;
    static constexpr int kPitch = kRowBytes + 16;                  // 16 more: no two of the rows read together share a bank
    static constexpr int kBytes = kKeys * kPitch;
    static constexpr int kStages = !INT8 && kKeys * DIM > 64 * 64 ? 2 : 3;         // the large ones as many as leave room for two blocks on an SM
    static constexpr int kStage = 2 * kBytes + (INT8 ? 2 * kKeys * 4 : 0);
    static constexpr int kJoin = kWarps * 16 * (DIM + 4) * 4;      // the warps' parts, where they share the keys
    static constexpr int kShared = kStages * kStage > kJoin ? kStages * kStage : kJoin;
};
template <int DIM, bool INT8, bool A, bool B> constexpr int shared_of() {
    return Tile<DIM, INT8, A>::kShared > Tile<DIM, INT8, B>::kShared ? Tile<DIM, INT8, A>::kShared : Tile<DIM, INT8, B>::kShared;
}

// of the threads that attend, in whatever block
__device__ __forceinline__ void attend_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }

// Rows of a tile: 16 to a warp (BY_KEYS false: 64 rows, every warp walks all keys) or the same 16 for all warps (BY_KEYS: a
// quarter of every tile of keys each, joined at the end), for the few rows of one sequence.
// What bounds it: one step's wait for the next (loads, products, exponentials) of three to four blocks on an SM.  128 sequences of up to 1025
// positions, 8 heads of 64: 134 MB in 30 us, 4.5 TB/s, two thirds of what HBM copies at.
template <int DIM, bool INT8, bool BY_KEYS>
__device__ __forceinline__ void attend(const PrefixParams& p, const Keys& keys, uint8_t* smem, int b, int g, int row_tile, int split, bool own) {
    using L = Tile<DIM, INT8, BY_KEYS>;
    constexpr int KEYS = L::kKeys, ROWS = BY_KEYS ? 16 : 16 * kWarps, NT = BY_KEYS ? KEYS / 8 / kWarps : KEYS / 8, COLS = DIM / 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, t4 = lane & 3;
    const int rows = own ? p.time * p.group : p.batch * p.time * p.group, row0 = row_tile * ROWS + (BY_KEYS ? 0 : 16 * warp);
    // This lane's two rows: where they lie among all rows, and their queries.  All that can be asked for at once is: the length and the queries, and behind
    // the length the first tiles, ahead of the queries' first use (under load each takes 1500 cycles; one after the other an item began at 6000).
    const int held = keys.lengths[b];
    long long at[2];
    int step[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int m = row0 + quad + 8 * i;
        step[i] = (int)((unsigned)m / (unsigned)p.group);
        at[i] = m < rows ? (((own ? (long long)b * p.time : 0) + step[i]) * p.kv_heads + g) * p.group + (m - step[i] * p.group) : -1;
    }
    uint32_t qf[DIM / 16][4];
#pragma unroll
    for (int kk = 0; kk < DIM / 16; ++kk)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // a lane's four elements of 16: two and two eight apart as the instruction numbers them; for 8-bit keys they are four
            // neighbours instead (one word of the key), the same permutation of the contraction on both sides
            const __nv_bfloat16* src = p.q + (at[i] < 0 ? 0 : at[i]) * DIM + kk * 16;
            uint2 v = make_uint2(0u, 0u);
            if (at[i] >= 0) {
                if (INT8) v = *reinterpret_cast<const uint2*>(src + 4 * t4);
                else v = make_uint2(*reinterpret_cast<const uint32_t*>(src + 2 * t4), *reinterpret_cast<const uint32_t*>(src + 2 * t4 + 8));
            }
            qf[kk][i] = v.x;
            qf[kk][2 + i] = v.y;
        }
    const int length = min(max(held, 0), keys.longest);
    const int begin = split * keys.chunk, end = min(length, begin + keys.chunk);
    int limit[2];                        // keys that the two rows see
#pragma unroll
    for (int i = 0; i < 2; ++i) limit[i] = at[i] < 0 ? 0 : own ? min(end, length - p.time + step[i] + 1) : end;

    const uint32_t base = smem_u32(smem);
    const long long head = ((own ? (long long)b * p.kv_heads : 0) + g) * keys.capacity;
    // a thread copies piece `piece` of every TOGETHER-th key of a tile
    constexpr int PIECES = L::kRowBytes / 16, TOGETHER = kThreads / PIECES;
    const int mine = threadIdx.x / PIECES, piece = threadIdx.x % PIECES;
    const long long from = (head + begin + mine) * L::kRowBytes + piece * 16;
    const uint32_t to = base + mine * L::kPitch + piece * 16;
    auto fetch = [&](int tile, int slot) {         // keys begin + KEYS tile ..; behind `end` zeros, whatever lies there
        const uint32_t stage = to + slot * L::kStage;
        const long long at = from + (long long)tile * KEYS * L::kRowBytes;
        const int left = end - begin - tile * KEYS - mine;
#pragma unroll
        for (int i = 0; i < KEYS / TOGETHER; ++i) {
            const bool there = i * TOGETHER < left;
            const long long src = there ? at + i * TOGETHER * L::kRowBytes : 0;
            copy16(stage + i * TOGETHER * L::kPitch, keys.k + src, there);
            copy16(stage + L::kBytes + i * TOGETHER * L::kPitch, keys.v + src, there);
        }
        if (INT8) {
#pragma unroll
            for (int i = threadIdx.x; i < 2 * KEYS; i += kThreads) {
                const int key = i & (KEYS - 1);
                const bool there = begin + tile * KEYS + key < end;
                copy4(base + slot * L::kStage + 2 * L::kBytes + i * 4, (i >= KEYS ? keys.v_scale : keys.k_scale) + (there ? head + begin + tile * KEYS + key : 0), there);
            }
        }
    };

    float o[COLS][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < COLS; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
    const int tiles = end > begin ? (end - begin + KEYS - 1) / KEYS : 0;
    const float scale2 = p.scale * LOG2E;
#pragma unroll
    for (int s = 0; s < L::kStages - 1; ++s) {
        if (s < tiles) fetch(s, s);
        copies_commit();
    }
    int slot = 0, ahead = L::kStages - 1;          // of tile j, of the one that is fetched
    // rows quad + 8 of a warp's 16, where there are so many
    const bool upper = rows - row0 > 8;
    for (int j = 0; j < tiles; ++j) {
        copies_wait<L::kStages - 2>();
        attend_sync();                 // tile j is here, and nobody reads the stage that is filled next
        if (j + L::kStages - 1 < tiles) fetch(j + L::kStages - 1, ahead);
        copies_commit();
        const uint32_t k_tile = base + slot * L::kStage, v_tile = k_tile + L::kBytes, scales = k_tile + 2 * L::kBytes;
        const int key0 = BY_KEYS ? warp * (KEYS / kWarps) : 0, first = begin + j * KEYS + key0;
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
        if (++slot == L::kStages) slot = 0;
        if (++ahead == L::kStages) ahead = 0;
        float alpha[2] = {1.f, 1.f}, from2[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (i && !upper) break;
            float peak = -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; ++n) peak = fmaxf(peak, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
            // the base of the exponentials follows the maximum only when it is 2^8 behind (see prefix_tensor_kernel)
            if (peak * scale2 > m[i] + 8.f) {
                alpha[i] = exp2_fast(m[i] - peak * scale2);
                m[i] = peak * scale2;
                l[i] *= alpha[i];
            }
            from2[i] = m[i] == -INFINITY ? 0.f : m[i];       // a row that has seen nothing yet
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                o[c][0] *= alpha[0]; o[c][1] *= alpha[0];
                o[c][2] *= alpha[1]; o[c][3] *= alpha[1];
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float2 vs = make_float2(1.f, 1.f);
            if constexpr (INT8) vs = load_shared_f2(scales + (KEYS + key0 + 8 * n + 2 * t4) * 4);      // the value's scale goes with its probability
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (i && !upper) {
                    s[n][2] = s[n][3] = 0.f;
                    break;
                }
                const float p0 = exp2_fast(fmaf(s[n][2 * i], scale2, -from2[i])), p1 = exp2_fast(fmaf(s[n][2 * i + 1], scale2, -from2[i]));
                l[i] += p0 + p1;
                s[n][2 * i] = INT8 ? p0 * vs.x : p0;
                s[n][2 * i + 1] = INT8 ? p1 * vs.y : p1;
            }
        }
#pragma unroll
        for (int ks = 0; ks < NT / 2; ++ks) {
            // probabilities as two bf16 numbers each, what one leaves in the other: 2^-16 of them is lost at most, so that the output's own rounding
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
        attend_sync();
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
        attend_sync();
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
            factor[w] = exp2_fast(part[(w * 16 + r) * (DIM + 4) + DIM] - from);
            total += factor[w] * part[(w * 16 + r) * (DIM + 4) + DIM + 1];
        }
        const bool whole = p.slots == 1;
        const long long slot = (long long)(keys.first_slot + split) * p.rows + to;
        const float inverse = total != 0.f ? 1.f / total : 0.f;         // (NaN stays)
        if (piece == 0) {
            if (whole) p.lse[to] = total != 0.f ? (top + log2f(total)) * LN2 : -INFINITY;
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
            const float inverse = l[i] != 0.f ? 1.f / l[i] : 0.f;
            if (t4 == 0) {
                if (p.slots == 1) p.lse[at[i]] = l[i] != 0.f ? (m[i] + log2f(l[i])) * LN2 : -INFINITY;
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

// ------------------------------------------------------------------------------------------------
// The prefix on the tcgen05 tensor cores, for rows that fill their tiles: 128 rows (whole groups of heads of 128 / group sequences) against
// blocks of 64 keys.  Warp 0 asks TMA for the tiles, warp 1 issues the MMAs, four row warps own a TMEM lane (a row) per thread:
//     S = Q K^T -> rows: max, exp2, sum, P as two bf16 numbers, put back over the scores -> O += P V, twice, accumulated in tensor memory.
// The scores of the next blocks go to other buffers meanwhile.  Keys and values of 8 bits come through warp 0 and two more, which load them
// and put them into shared memory as bf16, exactly, in the order in which TMA would have; their scales go to the rows, the key's into
// the score, the value's into the probability.
// What bounds it: the exponential unit, 512 cycles for a block (the products take 384, 256 of them the two of P V), beside the rows' other
// instructions; two CTAs to an SM, so that one's run beside the other's waits.  512 rows of 8 heads by 32768 keys of 64: 68 us, 1550 cycles for a block of each
// of the two CTAs, the exponential unit busy for 52 % of the time, the tensor cores for 39 %.  Three CTAs to an SM and more tiles ahead were no faster.
// ------------------------------------------------------------------------------------------------
constexpr int kTcKeys = 64, kTcColumns = 256, kTcConverters = 3;

template <int DIM, bool INT8> struct TcTile {
    static constexpr int kThreads = 192 + (INT8 ? 32 * (kTcConverters - 1) : 0);       // warp 0 is one of them
    static constexpr int kHalves = DIM / 64;                       // a row of 64 elements is the 128 bytes of a swizzle
    static constexpr int kQHalf = 128 * 128, kKeyHalf = kTcKeys * 128;
    static constexpr int kQ = kHalves * kQHalf, kKey = kHalves * kKeyHalf;
    static constexpr int kStages = DIM == 64 ? 3 : 2;
    static constexpr int kBuffers = DIM == 64 ? 3 : 2;             // of scores: with O all of a CTA's 256 columns
    static constexpr int kTiles = kQ + 2 * kStages * kKey;
    static constexpr int kScales = INT8 ? kStages * 2 * kTcKeys * 4 : 0;
    static constexpr int kNeeded = kTiles + 256 + kScales, kShared = kNeeded > shared_of<DIM, INT8, true, false>() ? kNeeded : shared_of<DIM, INT8, true, false>();
};

struct alignas(64) PrefixTcParams {
    CUtensorMap map_q, map_k, map_v;     // k, v: of a bf16 prefix
    PrefixParams p;
    int* status;
    int sequences;                       // of batch * time, in a tile
};

// 16 signed bytes as 16 bf16 numbers, to two neighbouring pieces of a swizzled row
__device__ __forceinline__ void store_bytes(uint32_t row, int piece, int key, const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t a = bytes_to_bf16(__byte_perm(w[2 * i], 0, 0x4140)), b = bytes_to_bf16(__byte_perm(w[2 * i], 0, 0x4342));
        const uint32_t c = bytes_to_bf16(__byte_perm(w[2 * i + 1], 0, 0x4140)), d = bytes_to_bf16(__byte_perm(w[2 * i + 1], 0, 0x4342));
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + (((2 * piece + i) ^ (key & 7)) << 4)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
    }
}

// The blocks behind the prefix's items see the sequences' own caches, as in prefix_attention_kernel, one launch for both.
template <int DIM, bool INT8, bool OWN_BY_KEYS>
__global__ void __launch_bounds__(TcTile<DIM, INT8>::kThreads, 2)
prefix_tensor_kernel(const __grid_constant__ PrefixTcParams tc) {
    using L = TcTile<DIM, INT8>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const PrefixParams& p = tc.p;
    if ((int)blockIdx.x >= p.prefix_items) {
        chain_wait();
        chain_next();
        if (threadIdx.x >= kThreads) return;
        const int item = (int)blockIdx.x - p.prefix_items, split = item % p.own.splits, tile = item / p.own.splits, head = tile / p.own.row_tiles;
        attend<DIM, INT8, OWN_BY_KEYS>(p, p.own, smem_raw, head / p.kv_heads, head % p.kv_heads, tile % p.own.row_tiles, split, true);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = (int)blockIdx.x % p.prefix.splits, tile = (int)blockIdx.x / p.prefix.splits;
    const int g = tile % p.kv_heads, first_sequence = tile / p.kv_heads * tc.sequences;
    const uint32_t base = smem_u32(smem_raw), q_tile = base, k_tile = base + L::kQ, v_tile = k_tile + L::kStages * L::kKey, bars = base + L::kTiles;
    enum { Q_FULL = 0, K_FULL = 1, V_FULL = K_FULL + L::kStages, K_EMPTY = V_FULL + L::kStages, V_EMPTY = K_EMPTY + L::kStages, S_FULL = V_EMPTY + L::kStages,
           P_FULL = S_FULL + L::kBuffers, BARS = P_FULL + L::kBuffers };
    static_assert(8 * BARS + 8 <= 256, "the barriers fit");
    float* const scales = reinterpret_cast<float*>(smem_raw + L::kTiles + 256);      // INT8: [stage][key, value][64]
    auto bar = [&](int which) { return bars + 8u * which; };
    uint32_t& s_tmem_base = *reinterpret_cast<uint32_t*>(smem_raw + L::kTiles + 8 * BARS);
    volatile int& s_abort = *reinterpret_cast<volatile int*>(smem_raw + L::kTiles + 8 * BARS + 4);
    if (base & 1023u) {                  // the operand tiles need the alignment the declaration asks for
        chain_wait();
        if (threadIdx.x == 0) atomicExch(tc.status, STATUS_ATTENTION_WAIT + 1);
        return;
    }
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int w = 0; w < BARS; ++w) mbar_init(bar(w), w >= P_FULL ? 4 : INT8 && w >= K_FULL && w < K_EMPTY ? kTcConverters : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&tc.map_q);
        if (!INT8) { prefetch_map(&tc.map_k); prefetch_map(&tc.map_v); }
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(kTcColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    chain_wait();
    chain_next();                        // the tensor memory is this block's
    const uint32_t tmem = s_tmem_base, tmem_o = tmem + L::kBuffers * kTcKeys;      // the buffers of scores, O behind them
    const int length = min(max(p.prefix.lengths[0], 0), p.prefix.longest);
    const int begin = split * p.prefix.chunk, end = min(length, begin + p.prefix.chunk);
    const int n = end > begin ? (end - begin + kTcKeys - 1) / kTcKeys : 0;
    const Wait wait{&s_abort, tc.status};

    if (warp == 0 && lane == 0 && n) {
        mbar_expect_tx(bar(Q_FULL), p.group * tc.sequences * DIM * 2);
        for (int half = 0; half < L::kHalves; ++half) tma_load_3d(&tc.map_q, q_tile + half * L::kQHalf, bar(Q_FULL), half * 64, g * p.group, first_sequence);
    }
    __syncwarp();
    if (INT8 && (warp == 0 || warp >= 6)) {
        // pieces of 16 values, a thread's EACH of a tile: piece i of the tile is piece i % PIECES of key i / PIECES
        constexpr int PIECES = DIM / 16, ALL = kTcKeys * PIECES, EACH = (ALL + 32 * kTcConverters - 1) / (32 * kTcConverters);
        const int mine = warp ? threadIdx.x - 160 : lane;
        const long long head = (long long)g * p.prefix.capacity + begin;
        uint4 k[EACH], v[EACH];
        float k_scale = 0.f, v_scale = 0.f;
        auto fetch = [&](int j) {        // behind `end` zeros, whatever lies there
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int at = i * 32 * kTcConverters + mine, key = j * kTcKeys + at / PIECES;
                const bool there = at < ALL && begin + key < end;
                const long long from = (head + key) * DIM + at % PIECES * 16;
                k[i] = there ? *reinterpret_cast<const uint4*>(p.prefix.k + from) : make_uint4(0, 0, 0, 0);
                v[i] = there ? *reinterpret_cast<const uint4*>(p.prefix.v + from) : make_uint4(0, 0, 0, 0);
            }
            const bool there = mine < kTcKeys && begin + j * kTcKeys + mine < end;
            k_scale = there ? p.prefix.k_scale[head + j * kTcKeys + mine] : 0.f;
            v_scale = there ? p.prefix.v_scale[head + j * kTcKeys + mine] : 0.f;
        };
        if (n) fetch(0);
        int st = 0;
        uint32_t parity = 1;
        bool ok = true;
        for (int j = 0; ok && j < n; ++j) {
            auto put = [&](uint32_t to, const uint4* values) {
#pragma unroll
                for (int i = 0; i < EACH; ++i) {
                    const int at = i * 32 * kTcConverters + mine, key = at / PIECES, piece = at % PIECES;
                    if (at < ALL) store_bytes(to + piece / 4 * L::kKeyHalf + key * 128, piece % 4, key, values[i]);
                }
            };
            ok = wait.all(bar(K_EMPTY + st), parity);
            if (!ok) break;
            put(k_tile + st * L::kKey, k);
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(K_FULL + st));
            ok = wait.all(bar(V_EMPTY + st), parity);
            if (!ok) break;
            put(v_tile + st * L::kKey, v);
            if (mine < kTcKeys) {
                scales[st * 2 * kTcKeys + mine] = k_scale;
                scales[st * 2 * kTcKeys + kTcKeys + mine] = v_scale;
            }
            if (j + 1 < n) fetch(j + 1);
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(V_FULL + st));
            if (++st == L::kStages) { st = 0; parity ^= 1u; }
        }
    } else if (warp == 0) {
        if (lane == 0) {
            int st = 0;
            uint32_t parity = 1;
            for (int j = 0; j < n && !s_abort; ++j) {
                if (!wait(bar(K_EMPTY + st), parity)) break;
                mbar_expect_tx(bar(K_FULL + st), L::kKey);
                for (int half = 0; half < L::kHalves; ++half)
                    tma_load_3d(&tc.map_k, k_tile + st * L::kKey + half * L::kKeyHalf, bar(K_FULL + st), half * 64, begin + j * kTcKeys, g);
                if (!wait(bar(V_EMPTY + st), parity)) break;
                mbar_expect_tx(bar(V_FULL + st), L::kKey);
                for (int half = 0; half < L::kHalves; ++half)
                    tma_load_3d(&tc.map_v, v_tile + st * L::kKey + half * L::kKeyHalf, bar(V_FULL + st), half * 64, begin + j * kTcKeys, g);
                if (++st == L::kStages) { st = 0; parity ^= 1u; }
            }
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc_s = make_idesc<false, false, 128>(kTcKeys), idesc_o = make_idesc<false, true, 128>(64);
        // descriptors of the first tiles; an offset in bytes goes into their address field in units of 16
        const uint64_t q_desc = make_desc(q_tile, 16, 1024), k_desc = make_desc(k_tile, 16, 1024), v_desc = make_desc(v_tile, 8192, 1024);
        auto scores = [&](int j) {       // S = Q K^T of block j into its buffer
            const int st = j % L::kStages;
            if (!wait.all(bar(K_FULL + st), (uint32_t)(j / L::kStages) & 1u)) return false;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t k_at = k_desc + (uint32_t)(st * (L::kKey >> 4));
                const uint32_t to = tmem + (uint32_t)(j % L::kBuffers) * kTcKeys;
#pragma unroll
                for (int kk = 0; kk < DIM / 16; ++kk)
                    umma_bf16(to, q_desc + ((kk / 4 * L::kQHalf + kk % 4 * 32) >> 4), k_at + ((kk / 4 * L::kKeyHalf + kk % 4 * 32) >> 4), idesc_s, kk ? 1u : 0u);
                umma_commit(bar(S_FULL + j % L::kBuffers));
                umma_commit(bar(K_EMPTY + st));
            }
            __syncwarp();
            return true;
        };
        // the scores are formed as many blocks ahead as there are buffers but one
        bool ok = n && wait.all(bar(Q_FULL), 0);
        for (int j = 0; ok && j < L::kBuffers - 1 && j < n; ++j) ok = scores(j);
        for (int j = 0; ok && j < n; ++j) {
            const int st = j % L::kStages, next = j + L::kBuffers - 1;
            // into the buffer of the block before, once the product that reads its P there is done
            if (j > 0) ok = wait.all(bar(V_EMPTY + (j - 1) % L::kStages), (uint32_t)((j - 1) / L::kStages) & 1u);
            if (ok && next < n) ok = scores(next);
            if (ok) ok = wait.all(bar(V_FULL + st), (uint32_t)(j / L::kStages) & 1u);
            if (ok) ok = wait.all(bar(P_FULL + j % L::kBuffers), (uint32_t)(j / L::kBuffers) & 1u);
            if (!ok) break;
            tc_fence_after();
            // O += P V, the larger part of P and what it left: P from tensor memory, V as it lies in memory (rows = keys) is the
            // MN-major operand
            if (elect_one()) {
                const uint64_t v_at = v_desc + (uint32_t)(st * (L::kKey >> 4));
                const uint32_t from = tmem + (uint32_t)(j % L::kBuffers) * kTcKeys;
#pragma unroll
                for (int kk = 0; kk < kTcKeys / 16; ++kk)
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int half = 0; half < L::kHalves; ++half)
                            umma_bf16_ts(tmem_o + half * 64, from + kk / 2 * 32 + part * 16 + kk % 2 * 8, v_at + ((half * L::kKeyHalf + kk * 2048) >> 4), idesc_o, (j | kk | part) ? 1u : 0u);
                umma_commit(bar(V_EMPTY + st));
            }
            __syncwarp();
        }
        // the last commit has arrived before this CTA's shared memory can go to another one
        if (ok) wait.all(bar(V_EMPTY + (n - 1) % L::kStages), (uint32_t)((n - 1) / L::kStages) & 1u);
    } else {
        const int quad = warp & 3, row = quad * 32 + lane;
        const int sequence = first_sequence + row / p.group;
        const bool live = row < p.group * tc.sequences && sequence < p.batch * p.time;
        const long long at = ((long long)sequence * p.kv_heads + g) * p.group + row % p.group;
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
        // Scores in the exponent of 2.  x = s * scale2 - m with m, a maximum, rounded there: what that is off by is in numerator and sum alike.
        const float scale2 = p.scale * LOG2E;
        const uint64_t scale_pair = pair2(scale2, scale2);
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        int st = 0, buffer = 0;          // of the block, and how often they have come round
        uint32_t st_round = 0, buffer_round = 0;
        for (int j = 0; ok && j < n; ++j) {
            const int there = end - begin - j * kTcKeys;            // keys of the block
            const uint32_t tmem_s = tmem + (uint32_t)buffer * kTcKeys + lane_base;
            ok = wait.all(bar(S_FULL + buffer), buffer_round);
            if (ok && (INT8 || there < kTcKeys)) ok = wait.all(bar(V_FULL + st), st_round);
            if (!ok) break;
            tc_fence_after();
            uint32_t s[kTcKeys];
            tmem_ld32(tmem_s, s);
            tmem_ld32(tmem_s + 32, s + 32);
            tmem_ld_wait();
            if constexpr (INT8) {
                const float4* by = reinterpret_cast<const float4*>(scales + st * 2 * kTcKeys);
#pragma unroll
                for (int c = 0; c < kTcKeys; c += 4) {
                    const float4 f = by[c / 4];
                    float x[4];
                    unpair2(mul2(pair2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), pair2(f.x, f.y)), x[0], x[1]);
                    unpair2(mul2(pair2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), pair2(f.z, f.w)), x[2], x[3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[c + i] = __float_as_uint(x[i]);
                }
            }
            if (there < kTcKeys) {
#pragma unroll
                for (int c = 0; c < kTcKeys; ++c)
                    if (c >= there) s[c] = 0xff800000u;             // -inf
                if constexpr (!INT8) {
                    // Whatever lies behind the prefix must not meet a probability of zero as a NaN: its values become zeros.
                    for (int i = threadIdx.x - 64; i < L::kHalves * kTcKeys * 8; i += 128)
                        if (i / 8 % kTcKeys >= there)
                            *reinterpret_cast<uint4*>(smem_raw + (v_tile - base) + st * L::kKey + i / 8 / kTcKeys * L::kKeyHalf + i / 8 % kTcKeys * 128 + i % 8 * 16) = make_uint4(0, 0, 0, 0);
                    fence_async_shared();
                }
            }
            float peak4[4] = {__uint_as_float(s[0]), __uint_as_float(s[1]), __uint_as_float(s[2]), __uint_as_float(s[3])};
#pragma unroll
            for (int c = 4; c < kTcKeys; c += 2) peak4[(c >> 1) & 3] = max3(peak4[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
            const float next = fmaxf(max3(peak4[0], peak4[1], peak4[2]), peak4[3]) * scale2;
            // The base of the exponentials follows the maximum only when it is 2^8 behind: a new maximum somewhere in 32 rows comes with every other block,
            // and rescaling O for it took a fifth of the rows' time.  Probabilities up to 2^8 keep their relative precision in the two bf16 numbers.
            const bool moves = next > m + 8.f;
            const float alpha = moves && j ? exp2_fast(m - next) : 1.f;
            if (moves) m = next;
            const float from = m == -INFINITY ? 0.f : m;
            l *= alpha;
            if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                // O is whole once the product of the block before is done
                ok = wait.all(bar(V_EMPTY + (j - 1) % L::kStages), (uint32_t)((j - 1) / L::kStages) & 1u);
                if (!ok) break;
                tc_fence_after();
                const uint64_t alpha_pair = pair2(alpha, alpha);
#pragma unroll 1
                for (int e = 0; e < DIM; e += 16) {
                    uint32_t o[16];
                    tmem_ld16(tmem_o + lane_base + e, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 16; c += 2) {
                        float o0, o1;
                        unpair2(mul2(pair2(__uint_as_float(o[c]), __uint_as_float(o[c + 1])), alpha_pair), o0, o1);
                        o[c] = __float_as_uint(o0);
                        o[c + 1] = __float_as_uint(o1);
                    }
                    tmem_st16(tmem_o + lane_base + e, o);
                }
            }
            const uint64_t minus_m = pair2(-from, -from);
            uint64_t total2[2] = {0, 0};
            // 32 keys at a time, back over their scores: the larger parts of their probabilities, then the rest
#pragma unroll
            for (int h = 0; h < kTcKeys; h += 32) {
                uint32_t high[16], rest[16];
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    float x0, x1;
                    unpair2(fma2(pair2(__uint_as_float(s[h + c]), __uint_as_float(s[h + c + 1])), scale_pair, minus_m), x0, x1);
                    float p0 = exp2_fast(x0), p1 = exp2_fast(x1);
                    total2[(c >> 1) & 1] = add2(total2[(c >> 1) & 1], pair2(p0, p1));
                    if constexpr (INT8) {
                        const float2 f = *reinterpret_cast<const float2*>(scales + (st * 2 + 1) * kTcKeys + h + c);
                        unpair2(mul2(pair2(p0, p1), pair2(f.x, f.y)), p0, p1);
                    }
                    split2(p0, p1, high[c >> 1], rest[c >> 1]);
                }
                tmem_st16(tmem_s + h, high);
                tmem_st16(tmem_s + h + 16, rest);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(P_FULL + buffer));
            if (++st == L::kStages) { st = 0; st_round ^= 1u; }
            if (++buffer == L::kBuffers) { buffer = 0; buffer_round ^= 1u; }
            float t0, t1;
            unpair2(add2(total2[0], total2[1]), t0, t1);
            l += t0 + t1;
        }
        if (ok && n) ok = wait.all(bar(V_EMPTY + (n - 1) % L::kStages), (uint32_t)((n - 1) / L::kStages) & 1u);
        if (ok) {
            const bool whole = p.slots == 1;
            const long long slot = (long long)(p.prefix.first_slot + split) * p.rows + at;
            const float inverse = l != 0.f ? 1.f / l : 0.f;
            if (live) {
                if (whole) p.lse[at] = l != 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
                else p.part_ml[slot] = make_float2(m, l);
            }
            if (n || whole) {
                tc_fence_after();
                // 32 columns at a time through shared memory (the tiles are done with), so that the rows are written in pieces of 128 bytes and not by
                // a thread each.  (A short item spends a quarter of its time here either way: 3400 of 14000 cycles, 64 sequences, 4096 keys.)
                constexpr int PITCH = 36;
                float* const stage = reinterpret_cast<float*>(smem_raw + (k_tile - base)) + quad * 32 * PITCH;
                const float factor = n ? whole ? inverse : 1.f : 0.f;
#pragma unroll 1
                for (int e = 0; e < DIM; e += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem_o + lane_base + e, o);
                    tmem_ld_wait();
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        auto value = [&](int i) { return n ? __uint_as_float(o[c + i]) * factor : 0.f; };
                        *reinterpret_cast<float4*>(stage + lane * PITCH + c) = make_float4(value(0), value(1), value(2), value(3));
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int r = i * 4 + lane / 8;
                        const float4 v = *reinterpret_cast<const float4*>(stage + r * PITCH + lane % 8 * 4);
                        const long long to = __shfl_sync(0xffffffffu, live ? at : -1, r);
                        if (to < 0) continue;
                        if (whole) *reinterpret_cast<uint2*>(p.out + to * DIM + e + lane % 8 * 4) = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
                        else *reinterpret_cast<float4*>(p.part_o + ((long long)(p.prefix.first_slot + split) * p.rows + to) * DIM + e + lane % 8 * 4) = v;
                    }
                }
            }
        }
    }
    linger_after_abort(&s_abort);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTcColumns) : "memory");
    }
}

// A key that a row does not see has a probability of zero there, but zero times a NaN or an infinity is not.  So, of several new positions, a row that
// comes out as no numbers, and not by its scores, is done again: by one warp, a key to a lane, as the formula says it, with no value that the row
// does not see.  What the prefix gave it is taken from its parts.
template <int DIM>
__device__ __noinline__ void row_again(const PrefixParams& p, long long row) {
    const Keys& keys = p.own;
    const int lane = threadIdx.x & 31, heads = p.kv_heads * p.group, h = (int)(row % heads), b = (int)(row / heads / p.time), step = (int)(row / heads % p.time);
    const int limit = min(max(keys.lengths[b], 0), keys.longest) - p.time + step + 1;
    const long long head = ((long long)b * p.kv_heads + h / p.group) * keys.capacity;
    const bool int8 = keys.k_scale != nullptr;
    const float scale2 = p.scale * LOG2E;
    const __nv_bfloat16* const q = p.q + row * DIM;
    float m = -INFINITY, l = 0.f, o[DIM / 32] = {};
    auto rescale = [&](float next) {     // returns the base of the exponentials
        const float from = next == -INFINITY ? 0.f : next, alpha = exp2_fast(m - from);
        m = next;
        l *= alpha;
#pragma unroll
        for (int c = 0; c < DIM / 32; ++c) o[c] *= alpha;
        return from;
    };
    for (int first = 0; first < limit; first += 32) {
        const long long key = head + first + lane;
        const bool sees = first + lane < limit;
        float score = -INFINITY;
        if (sees) {
            score = 0.f;
            for (int d = 0; d < DIM; ++d)
                score = fmaf(__bfloat162float(q[d]), int8 ? (float)((const int8_t*)keys.k)[key * DIM + d] : __bfloat162float(((const __nv_bfloat16*)keys.k)[key * DIM + d]), score);
            score *= int8 ? keys.k_scale[key] * scale2 : scale2;
        }
        const float from = rescale(fmaxf(m, warp_max(score))), weight = sees ? exp2_fast(score - from) : 0.f;
        l += warp_sum(weight);
        for (int i = 0; i < 32 && first + i < limit; ++i) {
            const float w = __shfl_sync(0xffffffffu, weight, i) * (int8 ? keys.v_scale[head + first + i] : 1.f);
#pragma unroll
            for (int c = 0; c < DIM / 32; ++c) {
                const long long at = (head + first + i) * DIM + 32 * c + lane;
                o[c] = fmaf(w, int8 ? (float)((const int8_t*)keys.v)[at] : __bfloat162float(((const __nv_bfloat16*)keys.v)[at]), o[c]);
            }
        }
    }
    for (int slot = 0; slot < p.prefix.splits; ++slot) {
        const float2 ml = p.part_ml[slot * p.rows + row];
        if (ml.y == 0.f) continue;       // saw no key, its values were not written
        const float weight = exp2_fast(ml.x - rescale(fmaxf(m, ml.x)));
        l += weight * ml.y;
#pragma unroll
        for (int c = 0; c < DIM / 32; ++c) o[c] = fmaf(weight, p.part_o[(slot * p.rows + row) * DIM + 32 * c + lane], o[c]);
    }
    const float inverse = l != 0.f ? 1.f / l : 0.f;
    if (lane == 0) p.lse[row] = l != 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
#pragma unroll
    for (int c = 0; c < DIM / 32; ++c) p.out[row * DIM + 32 * c + lane] = __float2bfloat16_rn(o[c] * inverse);
}

// the same for rows that come in one part: a warp looks at one of them
template <int DIM>
__global__ void __launch_bounds__(kThreads)
prefix_check_kernel(const __grid_constant__ PrefixParams p) {
    chain_begin();
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    bool odd = false;
#pragma unroll
    for (int c = 0; c < DIM / 32; ++c) odd |= !(fabsf(__bfloat162float(p.out[row * DIM + 32 * c + lane])) < INFINITY);
    if (__any_sync(0xffffffffu, odd) && p.lse[row] == p.lse[row]) row_again<DIM>(p, row);
}

// The parts of a row: WARPS warps to a row, which take every WARPS-th part, their weights a lane each, eight parts' values on their way together, and
// meet in shared memory.  One warp to a row, four rows to a block, where that leaves enough warps or there is little to each; else eight: 16 rows in 97
// parts of 128 values take 26 us with one and 5 with eight, 4096 rows in 10 parts 5 and 12.  What bounds it is the wait for the parts, from L2.
template <int DIM, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? kThreads : 32 * WARPS)
prefix_join_kernel(const __grid_constant__ PrefixParams p) {
    chain_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = WARPS == 1 ? 0 : warp;
    const long long row = WARPS == 1 ? (long long)blockIdx.x * kWarps + warp : blockIdx.x;
    if (row >= p.rows) return;
    constexpr int LANES = DIM / 4, TOGETHER = 32 / LANES, DEEP = 8 / TOGETHER;        // lanes of a part's row, parts at a time, such loads in flight
    float top = -INFINITY, total = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int first = mine; first < p.slots; first += 32 * WARPS) {
        const int slot = first + lane * WARPS;
        const float2 ml = slot < p.slots ? p.part_ml[slot * p.rows + row] : make_float2(-INFINITY, 0.f);
        const float next = fmaxf(top, warp_max(ml.x)), from = next == -INFINITY ? 0.f : next, alpha = exp2_fast(top - from);
        const bool saw = ml.y != 0.f;    // else no key: its values were not written
        const unsigned seen = __ballot_sync(0xffffffffu, saw);
        const float factor = saw ? ml.y == ml.y ? exp2_fast(ml.x - from) : ml.y : 0.f;         // NaN where the part is
        top = next;
        total = total * alpha + warp_sum(factor * ml.y);
        sum.x *= alpha; sum.y *= alpha; sum.z *= alpha; sum.w *= alpha;
        const int many = min(32, (p.slots - first + WARPS - 1) / WARPS);
        for (int s = 0; s < many; s += TOGETHER * DEEP) {
            float4 v[DEEP];
            float f[DEEP];
#pragma unroll
            for (int i = 0; i < DEEP; ++i) {
                const int part = s + i * TOGETHER + lane / LANES;
                f[i] = __shfl_sync(0xffffffffu, factor, part);                    // 0 from `many` on
                v[i] = seen >> part & 1 ? *reinterpret_cast<const float4*>(p.part_o + ((first + part * WARPS) * p.rows + row) * DIM + lane % LANES * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int i = 0; i < DEEP; ++i) { sum.x += f[i] * v[i].x; sum.y += f[i] * v[i].y; sum.z += f[i] * v[i].z; sum.w += f[i] * v[i].w; }
        }
    }
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) {
        sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
        sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
        sum.z += __shfl_xor_sync(0xffffffffu, sum.z, o);
        sum.w += __shfl_xor_sync(0xffffffffu, sum.w, o);
    }
    if constexpr (WARPS > 1) {
        __shared__ float2 s_ml[WARPS];
        __shared__ float4 s_sum[WARPS][LANES];
        if (lane == 0) s_ml[warp] = make_float2(top, total);
        if (lane < LANES) s_sum[warp][lane] = sum;
        __syncthreads();
        if (warp) return;
        const float2 ml = lane < WARPS ? s_ml[lane] : make_float2(-INFINITY, 0.f);
        top = warp_max(ml.x);
        const float factor = exp2_fast(ml.x - (top == -INFINITY ? 0.f : top));
        total = warp_sum(factor * ml.y);
        sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = __shfl_sync(0xffffffffu, factor, w);
            const float4 v = s_sum[w][lane % LANES];
            sum.x += f * v.x; sum.y += f * v.y; sum.z += f * v.z; sum.w += f * v.w;
        }
    }
    const float inverse = total != 0.f ? 1.f / total : 0.f;
    if (lane < LANES) *reinterpret_cast<uint2*>(p.out + row * DIM + lane * 4) = make_uint2(pack2(sum.x * inverse, sum.y * inverse), pack2(sum.z * inverse, sum.w * inverse));
    if (lane == 0) p.lse[row] = total != 0.f ? (top + log2f(total)) * LN2 : -INFINITY;
    if (p.checks && total == total && __any_sync(0xffffffffu, !(fabsf(sum.x) < INFINITY && fabsf(sum.y) < INFINITY && fabsf(sum.z) < INFINITY && fabsf(sum.w) < INFINITY))) {
        __syncwarp();
        row_again<DIM>(p, row);
    }
}

struct Plan { Keys prefix, own; int slots; long long prefix_items, own_items; bool tensor, together, prefix_by_keys, own_by_keys; };

// Chunks of keys: as long as they leave four items to an SM, but not below two tiles.  (Two and three items to an SM were not compared with that.)
Plan plan_of(const qmoe_prefix_attention_t* a, const qmoe_cache_t* c) {
    Plan plan = {};
    const long long group = a->heads / c->kv_heads, own_rows = a->time * group, all_rows = c->batch * own_rows;
    // Tensor memory's kernel begins 3 us later and takes 128 rows for the price of one: it is ahead from some 8e5 pairs of a query row and a key on with
    // 64 values to a head, from 4e5 on with 128 (4 heads, without it and with it: 64 rows by 2048 keys 8.4 and 9.9 us, with 128 values 13.6 and 12.4;
    // 32 by 32768: 25 and 18, 41 and 22; 256 by 8192: 25 and 19, 39 and 24).  Up to 16 rows the other form has every warp at work on keys of its own and
    // stays ahead (8 heads of int8, 16 rows, 16384 keys: 22 us and 30), as it does for short prefixes (1024 rows of 8 heads by 256 keys: 34 and 40).
    plan.tensor = group <= 128 && all_rows > 16 && a->prefix_longest >= 512 && all_rows * c->kv_heads * c->dim * a->prefix_longest >= 50000000;
    plan.prefix_by_keys = all_rows <= 16;
    plan.own_by_keys = own_rows <= 16;
    plan.prefix.row_tiles = plan.tensor ? ceil_div(c->batch * a->time, 128 / group) : ceil_div(all_rows, plan.prefix_by_keys ? 16 : 64);
    plan.own.row_tiles = ceil_div(own_rows, plan.own_by_keys ? 16 : 64);
    const long long prefix_tiles = ceil_div(a->prefix_longest, kKeys), own_tiles = ceil_div(a->longest, kKeys), wanted = (long long)sm_count() * 4;
    const long long prefix_heads = (long long)plan.prefix.row_tiles * c->kv_heads, own_heads = (long long)plan.own.row_tiles * c->kv_heads * c->batch;
    const long long prefix_mma = plan.tensor ? 0 : prefix_tiles;
    long long chunk = prefix_mma > own_tiles ? prefix_mma : own_tiles;
    auto items = [&](long long tiles) { return prefix_heads * ceil_div(prefix_mma, tiles) + own_heads * ceil_div(own_tiles, tiles); };
    while (chunk > 2 && items(chunk) < wanted) chunk = (chunk + 1) / 2;
    if (chunk < 1) chunk = 1;
    plan.prefix.chunk = plan.own.chunk = (int)chunk * kKeys;
    if (plan.tensor) {                   // one round of the two CTAs that an SM holds, but no chunk below four blocks
        long long splits = 2ll * sm_count() / prefix_heads;
        if (splits > prefix_tiles / 4) splits = prefix_tiles / 4;
        plan.prefix.chunk = ceil_div(prefix_tiles, splits > 1 ? splits : 1) * kKeys;
    }
    plan.prefix.splits = ceil_div(a->prefix_longest, plan.prefix.chunk);
    plan.own.splits = ceil_div(own_tiles, chunk);
    if (!plan.prefix.splits && !plan.own.splits) plan.own.splits = 1;        // nothing to see: zeros are written all the same
    plan.own.first_slot = plan.prefix.splits;
    plan.slots = plan.prefix.splits + plan.own.splits;
    plan.prefix_items = prefix_heads * plan.prefix.splits;
    plan.own_items = own_heads * plan.own.splits;
    // One launch for both while the sequences' items are few.  Many of them are better off with a launch of their own, whose blocks are small and
    // three to four on an SM.  In one launch and in two, 4 or 8 key/value heads over prefixes of 1003 to 32768 keys: 78 items 13.6 and 22.8 us, 256 19.7 and 19.2,
    // 384 16.6 and 17.4, 592 33.0 and 32.8, 800 36.5 and 31.3, 888 37.6 and 31.0, 1024 30.5 and 24.9 (another such 128 and 114).
    plan.together = plan.own_items <= 4ll * sm_count();
    return plan;
}

void keys_of(const qmoe_cache_t* c, long long longest, Keys& k) {
    k.k = (const uint8_t*)c->k; k.v = (const uint8_t*)c->v;
    if (c->dtype == QMOE_INT8) { k.k_scale = (const float*)c->k_scale; k.v_scale = (const float*)c->v_scale; }
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

template <int DIM, bool INT8, bool OWN_BY_KEYS>
int launch_tensor(const PrefixParams& p, const Plan& plan, const qmoe_cache_t* prefix, cudaStream_t stream) {
    using L = TcTile<DIM, INT8>;
    PrefixTcParams tc = {};
    const uint32_t group = (uint32_t)p.group, sequences = 128 / group;
    if (int rc = make_map_3d(&tc.map_q, (uint64_t)p.q, DIM, (uint64_t)group * p.kv_heads, (uint64_t)p.batch * p.time, group, sequences)) return rc;
    if (!INT8) {
        if (int rc = make_map_3d(&tc.map_k, prefix->k, DIM, (uint64_t)prefix->capacity, (uint64_t)p.kv_heads, kTcKeys)) return rc;
        if (int rc = make_map_3d(&tc.map_v, prefix->v, DIM, (uint64_t)prefix->capacity, (uint64_t)p.kv_heads, kTcKeys)) return rc;
    }
    tc.p = p;
    tc.status = device_status_address();
    tc.sequences = (int)sequences;
    QMOE_CUDA((allow_shared<prefix_tensor_kernel<DIM, INT8, OWN_BY_KEYS>>(L::kShared)));
    chained(prefix_tensor_kernel<DIM, INT8, OWN_BY_KEYS>, (unsigned)(plan.prefix_items + (plan.together ? plan.own_items : 0)), L::kThreads, L::kShared, stream, tc);
    count_tensor_core_launch();
    QMOE_LAUNCH_CHECK("prefix_tensor_kernel");
    return 0;
}

template <int DIM, bool INT8>
int launch(PrefixParams& p, const Plan& plan, const qmoe_cache_t* prefix, cudaStream_t stream) {
    long long items = plan.prefix_items + plan.own_items;
    if (plan.tensor) {
        if (int rc = plan.own_by_keys ? launch_tensor<DIM, INT8, true>(p, plan, prefix, stream) : launch_tensor<DIM, INT8, false>(p, plan, prefix, stream)) return rc;
        items = plan.together ? 0 : plan.own_items;
        p.prefix_items = 0;
    }
    auto go = [&](auto prefix_by_keys, auto own_by_keys) -> int {
        constexpr bool A = decltype(prefix_by_keys)::value, B = decltype(own_by_keys)::value;
        constexpr int SHARED = shared_of<DIM, INT8, A, B>();
        QMOE_CUDA((allow_shared<prefix_attention_kernel<DIM, INT8, A, B>>(SHARED)));
        chained(prefix_attention_kernel<DIM, INT8, A, B>, (unsigned)items, kThreads, SHARED, stream, p);
        QMOE_LAUNCH_CHECK("prefix_attention_kernel");
        return 0;
    };
    int rc = 0;
    if (!items) {}
    else if (plan.own_by_keys && (plan.tensor || plan.prefix_by_keys)) rc = go(std::true_type(), std::true_type());
    else if (plan.own_by_keys) rc = go(std::false_type(), std::true_type());
    else rc = go(std::false_type(), std::false_type());
    if (rc) return rc;
    if (plan.slots == 1) {
        if (!p.checks) return 0;
        chained(prefix_check_kernel<DIM>, (unsigned)((p.rows + kWarps - 1) / kWarps), kThreads, 0, stream, p);
        QMOE_LAUNCH_CHECK("prefix_check_kernel");
        return 0;
    }
    if (plan.slots <= 8 || plan.slots * 32 <= p.rows) chained(prefix_join_kernel<DIM, 1>, (unsigned)((p.rows + kWarps - 1) / kWarps), kThreads, 0, stream, p);
    else chained(prefix_join_kernel<DIM, 8>, (unsigned)p.rows, 256, 0, stream, p);
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
    p.checks = a->time > 1 && a->longest > 0 && a->out != a->q;      // (queries that are being written over cannot be read again)
    if (c->dim == 64) return c->dtype == QMOE_INT8 ? launch<64, true>(p, plan, prefix, stream) : launch<64, false>(p, plan, prefix, stream);
    return c->dtype == QMOE_INT8 ? launch<128, true>(p, plan, prefix, stream) : launch<128, false>(p, plan, prefix, stream);
}
