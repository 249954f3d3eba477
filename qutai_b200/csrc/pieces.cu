// Softmax cross entropy over a vocabulary without keeping its logits, and its gradient:
//     loss = mean over the rows that have a target of  log sum_c exp(h_r . w_c) - h_r . w_target(r),
//     d h_r = sum_c g[r, c] w_c,   d w_c = sum_r g[r, c] h_r,   g[r, c] = (softmax(r)[c] - [c = target(r)]) x gradient / counted rows.
// The head that keeps its logits (head.cu) holds rows x vocab of them from the forward to the backward: 2 GB for 8192 rows of 131072
// classes.  Here the forward keeps a number a row.
//   * Rows with a target are gathered once, in their order, and counted on the device: rows without one cost nothing in the products, and
//     whatever they hold enters no gradient.
//   * Forward: one product on the tensor cores (gemm_tcgen05.cu, MODE_LOSS) whose epilogue keeps each row's largest logit and its sum of exponentials over
//     128 columns, in fp32 from the accumulator, and the target's logit; the logits are never written.  The parts of a row meet in fp32 in a fixed order.
//   * Backward, for each piece of the vocabulary: the piece's logits again, left as softmax minus one-hot in bf16; the product with the table's piece added to
//     the hidden rows' gradient in fp32; the product with the hidden rows, which is the piece of the table's gradient.  The factor gradient / counted
//     rows is applied to the finished sums: before the rounding to bf16 it would shift every row's -1 by the same up to 2^-9 (a share of 32000 classes is
//     next to nothing beside it: d_hidden 0.0026 off in the 2-norm like that, 0.0017 like this).
// 8 R V d operations, one product more than the 6 R V d of a head that forms its logits once: the price of cutting the vocabulary, whose first pieces' gradients wait for the
// sums of all.  (Cut over the rows instead, a chunk's logits could become gradients at once, in three products: not built.)
// float32 rows (the parity mode) take the CUDA-core products, a piece of logits at a time in both directions.
// No atomics: the same inputs give the same bits.
#include "common.cuh"

#include <math.h>

namespace qmoe {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kGroup = 64;              // rows that are counted together
constexpr int kGather = 16;             // rows of a block of the gathering kernel

// what the device knows of the rows: i32 words behind one another in `tables`
struct Tables {
    int* offsets;       // [2] 0, counted rows rounded up to 128
    int* counts;        // [2] counted rows, 0
    float* factor;      // [4] 1 / counted rows (at least 1)
    int* groups;        // [ceil(rows / 64)] counted rows of each 64
    int* place;         // [rows] where a row went, -1 without a target
    int* labels;        // [bound] target of each gathered row
    float* picked;      // [bound] its logit
};
long long bound_of(long long rows) { return (rows + kRowPad - 1) / kRowPad * kRowPad; }
long long group_words(long long rows) { return (rows + kGroup - 1) / kGroup; }
Tables tables_of(const qmoe_pieces_t* a) {
    int* base = (int*)a->tables;
    Tables t;
    t.offsets = base; t.counts = base + 2; t.factor = (float*)(base + 4);
    t.groups = base + 8; t.place = t.groups + group_words(a->rows); t.labels = t.place + a->rows;
    t.picked = (float*)(t.labels + bound_of(a->rows));
    return t;
}

__device__ __forceinline__ bool is_class(long long target, long long vocab) { return target >= 0 && target < vocab; }

// a warp counts 64 rows
__global__ void __launch_bounds__(kThreads)
count_kernel(const long long* __restrict__ targets, long long rows, long long vocab, int* __restrict__ groups) {
    chain_begin();
    const long long group = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (group * kGroup >= rows) return;
    int n = 0;
#pragma unroll
    for (int u = 0; u < kGroup / 32; ++u) {
        const long long r = group * kGroup + u * 32 + lane;
        n += __popc(__ballot_sync(0xffffffffu, r < rows && is_class(targets[r], vocab)));
    }
    if (lane == 0) groups[group] = n;
}

// A block gathers 16 rows in 16-byte pieces, a warp two of them with their loads in flight, behind the counted rows before them; the last block knows how many
// there are, and clears the rows up to the next multiple of 16, which the products over rows read.
__global__ void __launch_bounds__(kThreads)
gather_kernel(const uint4* __restrict__ hidden, const long long* __restrict__ targets, uint4* __restrict__ inputs, Tables t, long long rows, long long vocab,
              long long pieces) {
    chain_begin();
    __shared__ int s_part[kWarps];
    __shared__ unsigned s_flags[kGroup / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long first = (long long)blockIdx.x * kGather, group = first / kGroup, group_row = group * kGroup;
    int before = 0;
    for (long long g = threadIdx.x; g < group; g += kThreads) before += t.groups[g];
#pragma unroll
    for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (lane == 0) s_part[warp] = before;
    if (warp < kGroup / 32) {
        const long long r = group_row + warp * 32 + lane;
        const unsigned flags = __ballot_sync(0xffffffffu, r < rows && is_class(targets[r], vocab));
        if (lane == 0) s_flags[warp] = flags;
    }
    __syncthreads();
    before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) before += s_part[w];
#pragma unroll
    for (int u = 0; u < kGather / kWarps; ++u) {
        const long long r = first + u * kWarps + warp;
        if (r >= rows) break;
        const int i = (int)(r - group_row);          // of its group's 64
        int at = before;
#pragma unroll
        for (int w = 0; w < kGroup / 32; ++w)
            at += __popc(w < i / 32 ? s_flags[w] : w == i / 32 ? s_flags[w] & ((1u << (i & 31)) - 1u) : 0u);
        const bool counted = s_flags[i / 32] >> (i & 31) & 1u;
        if (lane == 0) {
            t.place[r] = counted ? at : -1;
            if (counted) t.labels[at] = (int)targets[r];
        }
        if (!counted) continue;
        const uint4* from = hidden + r * pieces;
        uint4* to = inputs + at * pieces;
        for (long long c0 = 0; c0 < pieces; c0 += 32 * 8) {
            uint4 v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c0 + e * 32 + lane < pieces) v[e] = from[c0 + e * 32 + lane];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c0 + e * 32 + lane < pieces) to[c0 + e * 32 + lane] = v[e];
        }
    }
    if (blockIdx.x + 1 < gridDim.x) return;
    int all = before;
#pragma unroll
    for (int w = 0; w < kGroup / 32; ++w) all += __popc(s_flags[w]);
    if (threadIdx.x == 0) {
        t.offsets[0] = 0; t.offsets[1] = (all + kRowPad - 1) / kRowPad * kRowPad;
        t.counts[0] = all; t.counts[1] = 0;
        t.factor[0] = 1.f / (float)(all > 1 ? all : 1);
    }
    for (long long c = all * pieces + threadIdx.x; c < ((all + 15) & ~15) * pieces; c += kThreads) inputs[c] = make_uint4(0, 0, 0, 0);
}

// The parts of a row, largest logit and sum of exponentials against it, joined: 32 rows to a block, eight threads to a row.
__global__ void __launch_bounds__(kThreads)
join_kernel(const float2* __restrict__ statistics, long long pitch, int parts, Tables t, float* __restrict__ lse, float* __restrict__ row_loss) {
    chain_begin();
    __shared__ float2 s_part[kWarps][32];
    const int share = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long r = (long long)blockIdx.x * 32 + lane;
    const int count = t.counts[0];
    if ((long long)blockIdx.x * 32 >= count) return;
    float top = -INFINITY, total = 0.f;
    auto add = [&](float2 v) {
        const float higher = fmaxf(top, v.x), base = higher == -INFINITY ? 0.f : higher;
        total = total * expf(top - base) + v.y * expf(v.x - base);
        top = higher;
    };
    if (r < count) {
        int i = share;
        for (; i + 3 * kWarps < parts; i += 4 * kWarps) {
            float2 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = statistics[(long long)(i + u * kWarps) * pitch + r];
#pragma unroll
            for (int u = 0; u < 4; ++u) add(v[u]);
        }
        for (; i < parts; i += kWarps) add(statistics[(long long)i * pitch + r]);
    }
    s_part[share][lane] = make_float2(top, total);
    __syncthreads();
    if (share || r >= count) return;
    for (int w = 1; w < kWarps; ++w) add(s_part[w][lane]);
    const float log_sum = top + logf(total);
    lse[r] = log_sum;
    row_loss[r] = log_sum - t.picked[r];
}

// loss = sum of the row losses over their number, added in 64 bits in a fixed order
__global__ void __launch_bounds__(1024) mean_kernel(const float* __restrict__ row_loss, Tables t, float* __restrict__ loss) {
    chain_begin();
    __shared__ double s_sum[32];
    const int count = t.counts[0];
    double mine = 0.0;
    for (int r = threadIdx.x; r < count; r += 1024) mine += (double)row_loss[r];
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = mine;
    __syncthreads();
    if (threadIdx.x) return;
    double total = 0.0;
    for (int w = 0; w < 32; ++w) total += s_sum[w];
    loss[0] = (float)(total / (double)(count > 1 ? count : 1));
}

// d_hidden: the gathered rows' gradient, `parts` sums of it added in their order and times the factors, back in their places; zeros for rows without a
// target; a warp to a row
template <typename T>
__global__ void __launch_bounds__(kThreads)
scatter_kernel(const float* __restrict__ sum, int parts, long long part, const float* __restrict__ factor, const float* __restrict__ factor2, T* __restrict__ d_hidden,
               const int* __restrict__ place, long long rows, long long width) {
    chain_begin();
    constexpr int N = Vec16<T>::N;
    const long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int at = place[row];
    const float by = (factor ? factor[0] : 1.f) * (factor2 ? factor2[0] : 1.f);
    for (long long c = (threadIdx.x & 31) * N; c < width; c += 32 * N) {
        float v[N] = {};
        if (at >= 0) {
            for (int z = 0; z < parts; ++z) {
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(sum + z * part + at * width + c + i);
                    v[i] += x.x; v[i + 1] += x.y; v[i + 2] += x.z; v[i + 3] += x.w;
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] *= by;
        }
        *reinterpret_cast<uint4*>(d_hidden + row * width + c) = Vec16<T>::pack(v);
    }
}

// without a row that has a target nothing writes the table's gradient
__global__ void __launch_bounds__(kThreads) clear_unwritten_kernel(uint4* __restrict__ out, long long pieces, const int* __restrict__ counts) {
    chain_begin();
    if (counts[0]) return;
    for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < pieces; i += (long long)gridDim.x * kThreads) out[i] = make_uint4(0, 0, 0, 0);
}

// ---- float32 rows: a block to a row of a piece of logits ---------------------------------------------------------
__device__ __forceinline__ float block_join(float v, bool largest, float* tmp) {
    v = largest ? warp_max(v) : warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = tmp[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) r = largest ? fmaxf(r, tmp[w]) : r + tmp[w];
    return r;
}
// one part's statistics for the whole piece, and the target's logit
__global__ void __launch_bounds__(kThreads)
row_statistics_kernel(const float* __restrict__ logits, long long pitch, long long columns, long long first, Tables t, float2* __restrict__ statistics) {
    chain_begin();
    __shared__ float tmp[kWarps];
    const long long r = blockIdx.x;
    if (r >= t.counts[0]) return;
    const float* row = logits + r * pitch;
    float top = -INFINITY, total = 0.f;
    for (long long c = threadIdx.x; c < columns; c += kThreads) top = fmaxf(top, row[c]);
    top = block_join(top, true, tmp);
    const float base = top == -INFINITY ? 0.f : top;
    for (long long c = threadIdx.x; c < columns; c += kThreads) total += expf(row[c] - base);
    total = block_join(total, false, tmp);
    if (threadIdx.x) return;
    statistics[r] = make_float2(top, total);
    const long long label = t.labels[r] - first;
    if (label >= 0 && label < columns) t.picked[r] = row[label];
}
// in place; rows that are none (there are `gridDim.x` in the buffer) become zeros, which the products over rows read
__global__ void __launch_bounds__(kThreads)
row_gradient_kernel(float* __restrict__ logits, long long pitch, long long columns, long long first, Tables t, const float* __restrict__ lse, const float* __restrict__ gradient) {
    chain_begin();
    const long long r = blockIdx.x;
    float* row = logits + r * pitch;
    if (r >= t.counts[0]) {
        for (long long c = threadIdx.x; c < columns; c += kThreads) row[c] = 0.f;
        return;
    }
    const float scale = t.factor[0] * (gradient ? gradient[0] : 1.f), log_sum = lse[r];
    const long long label = t.labels[r] - first;
    for (long long c = threadIdx.x; c < columns; c += kThreads) row[c] = scale * (expf(row[c] - log_sum) - (c == label ? 1.f : 0.f));
}

// columns of the buffer of a piece's logits or their gradient, whose rows start on 16 bytes
long long pitch_of(const qmoe_pieces_t* a) { const long long n = a->piece < a->vocab ? a->piece : a->vocab; return (n + 7) / 8 * 8; }
// float32: the sums over a piece's classes cut in up to 32 parts of at least 256, side by side, as far as 128 MB of them go.  301 rows of 256, 5003 classes: 563 us in
// one part of 20 tiles, 38 in 20, and chains of a twentieth of the length.
// bf16: the hidden rows' gradient has few tiles and a long sum.  In as many parts as there are pairs of SMs for its tiles of 256 x 256, of at least eight blocks of 64 classes.
long long parts_of(const qmoe_pieces_t* a) {
    if (a->dtype == QMOE_BF16) {
        const long long tiles = (a->rows + 255) / 256 * ((a->width + 255) / 256), blocks = (pitch_of(a) + 511) / 512, side = 74 / tiles < 32 ? 74 / tiles : 32;
        return side < 1 ? 1 : side < blocks ? side : blocks;
    }
    const long long most = (128ll << 20) / (a->rows * a->width * 4), wanted = (pitch_of(a) + 255) / 256, parts = wanted < 32 ? wanted : 32;
    return most < 1 ? 1 : parts < most ? parts : most;
}
// where the second buffer in the scratch starts: the hidden rows' gradient, or (forward, float32) the rows' statistics
long long second_of(const qmoe_pieces_t* a) { return a->dtype == QMOE_F32 ? a->rows * pitch_of(a) * 4 : bound_of(a->rows) * pitch_of(a) * 2; }
long long scratch_of(const qmoe_pieces_t* a, bool backward) {
    const long long pieces = (a->vocab + a->piece - 1) / a->piece;
    if (a->dtype == QMOE_F32) return second_of(a) + (backward ? parts_of(a) * a->rows * a->width * 4 : a->rows * pieces * 8);
    return backward ? second_of(a) + parts_of(a) * bound_of(a->rows) * a->width * 4 : (a->vocab + 255) / 256 * 2 * bound_of(a->rows) * 8;
}

int pieces_check(const qmoe_pieces_t* a, bool backward) {
    if (!a) return fail_arg("pieces: argument is null");
    if (a->dtype != QMOE_BF16 && a->dtype != QMOE_F32) return fail_arg("pieces: dtype must be QMOE_F32 or QMOE_BF16");
    if (a->weight_gradient != QMOE_F32 && (a->weight_gradient != QMOE_BF16 || a->dtype != QMOE_BF16))
        return fail_arg("pieces: the table's gradient is QMOE_F32, or QMOE_BF16 beside bf16 rows");
    if (a->rows <= 0 || a->width <= 0 || a->vocab <= 0 || a->piece <= 0) return fail_arg("pieces: sizes must be positive");
    if (a->rows > 0x7fffff00ll || a->vocab > 0x7fffff00ll || a->width > (1 << 24) || a->piece % 256) return fail_arg("pieces: sizes beyond 32 bits, or a piece that is no multiple of 256");
    const long long item = a->dtype == QMOE_BF16 ? 2 : 4;
    if ((a->width * item) % 16) return fail_arg("pieces: a row of hidden must be a multiple of 16 bytes");
    if (!a->hidden || !a->weight || !a->targets || !a->tables || !a->inputs || !a->lse || !a->row_loss || !a->scratch) return fail_arg("pieces: null buffer address");
    if (!backward && !a->loss) return fail_arg("pieces: null buffer address");
    if (backward && !a->d_hidden && !a->d_weight) return fail_arg("pieces: nothing to compute");
    if ((a->hidden | a->weight | a->inputs | a->scratch | a->d_hidden | a->d_weight | a->tables) & 15u) return fail_arg("pieces: buffers must be 16-byte aligned");
    if (a->targets & 7u || (a->lse | a->row_loss | a->loss | a->gradient) & 3u) return fail_arg("pieces: misaligned address");
    // what a call writes lies apart from all it reads and from one another (hidden is not read by the backward, which has the gathered rows)
    struct Span { uint64_t at; long long bytes; };
    auto overlap = [](const Span& x, const Span& y) { return x.at && y.at && x.at < y.at + (uint64_t)y.bytes && y.at < x.at + (uint64_t)x.bytes; };
    const long long bound = bound_of(a->rows);
    const Span hidden = {a->hidden, a->rows * a->width * item}, weight = {a->weight, a->vocab * a->width * item}, targets = {a->targets, a->rows * 8};
    const Span tables = {a->tables, (8 + group_words(a->rows) + a->rows + 2 * bound) * 4}, inputs = {a->inputs, bound * a->width * item}, lse = {a->lse, bound * 4};
    const Span gradient = {backward ? a->gradient : 0, 4}, row_loss = {a->row_loss, bound * 4}, none = {0, 0};
    const Span scratch = {a->scratch, scratch_of(a, backward)};
    const auto forward = [&](const Span& x) { return backward ? none : x; };
    const auto kept = [&](const Span& x) { return backward ? x : none; };        // what the forward leaves is what the backward reads
    const Span written[7] = {{backward ? a->d_hidden : a->loss, backward ? a->rows * a->width * item : 4},
                             {backward ? a->d_weight : 0, a->vocab * a->width * (a->weight_gradient == QMOE_BF16 ? 2 : 4)},
                             scratch, forward(inputs), forward(tables), forward(lse), forward(row_loss)};
    const Span read[7] = {weight, targets, gradient, forward(hidden), kept(inputs), kept(tables), kept(lse)};
    for (int i = 0; i < 7; ++i) {
        for (const Span& other : read)
            if (overlap(written[i], other)) return fail_arg("pieces: an output overlaps an operand");
        for (int j = 0; j < i; ++j)
            if (overlap(written[i], written[j])) return fail_arg("pieces: two outputs overlap");
    }
    return 0;
}

SimtGemmArgs simt(uint64_t a, uint64_t b, uint64_t c, long long m, long long n, long long k) {
    SimtGemmArgs g = {};
    g.A = (const void*)a; g.B = (const void*)b; g.C = (void*)c;
    g.M = m; g.N = n; g.K = k; g.mode = SG_PLAIN; g.ldc = n;
    return g;
}
// logits [rows, columns] of classes [first, first + columns)
int float_logits(const qmoe_pieces_t* a, long long first, long long columns, uint64_t logits, cudaStream_t stream) {
    SimtGemmArgs g = simt(a->inputs, a->weight + first * a->width * 4, logits, a->rows, columns, a->width);
    g.a_rs = a->width; g.a_cs = 1; g.b_rs = 1; g.b_cs = a->width; g.ldc = pitch_of(a);
    return launch_simt_gemm(g, QMOE_F32, QMOE_F32, QMOE_F32, a->rows, 1, stream);
}
PieceGemm piece_gemm(const qmoe_pieces_t* a, const Tables& t, long long first, long long columns) {
    PieceGemm g = {};
    g.inputs = a->inputs; g.weight = a->weight + first * a->width * 2;
    g.rows = bound_of(a->rows); g.width = a->width; g.columns = columns; g.first = first; g.pitch = pitch_of(a);
    g.offsets = t.offsets; g.counts = t.counts; g.labels = t.labels; g.lse = (const float*)a->lse; g.factor = t.factor;
    g.factor2 = (const float*)a->gradient;
    g.statistics = (float*)a->scratch; g.picked = t.picked;
    return g;
}

}  // namespace
}  // namespace qmoe

using namespace qmoe;

extern "C" int64_t qmoe_pieces_table_words(int64_t rows) {
    return rows <= 0 ? 0 : 8 + group_words(rows) + rows + 2 * bound_of(rows);
}

extern "C" int64_t qmoe_pieces_scratch_bytes(const qmoe_pieces_t* a, int32_t backward) {
    return !a || a->rows <= 0 || a->width <= 0 || a->vocab <= 0 || a->piece <= 0 ? 0 : scratch_of(a, backward != 0);
}

extern "C" int qmoe_pieces_forward(const qmoe_pieces_t* a, uint64_t stream_) {
    if (int rc = pieces_check(a, false)) return rc;
    cudaStream_t stream = (cudaStream_t)stream_;
    const Tables t = tables_of(a);
    const long long item = a->dtype == QMOE_BF16 ? 2 : 4, bound = bound_of(a->rows), words = a->width * item / 16;
    const long long groups = group_words(a->rows);
    {
        TimedScope timed(KC_OTHER, stream);
        // float32: the products run over all rows of the buffer
        if (a->dtype == QMOE_F32) QMOE_CUDA(cudaMemsetAsync((void*)a->inputs, 0, (size_t)(a->rows * a->width * 4), stream));
        chained(count_kernel, (unsigned)ceil_div(groups, kWarps), kThreads, 0, stream, (const long long*)a->targets, a->rows, a->vocab, t.groups);
        QMOE_LAUNCH_CHECK("count_kernel");
        chained(gather_kernel, (unsigned)ceil_div(a->rows, kGather), kThreads, 0, stream, (const uint4*)a->hidden, (const long long*)a->targets, (uint4*)a->inputs, t, a->rows, a->vocab,
                words);
        QMOE_LAUNCH_CHECK("gather_kernel");
    }
    int parts = 0;
    long long pitch = bound;
    const float2* statistics = (const float2*)a->scratch;
    if (a->dtype == QMOE_BF16) {
        TimedScope timed(KC_EXPERT_GEMM, stream);
        if (int rc = tc_piece_statistics(piece_gemm(a, t, 0, a->vocab), stream)) return rc;
        parts = 2 * ceil_div(a->vocab, 256);
    } else {
        TimedScope timed(KC_EXPERT_GEMM, stream);
        float2* to = (float2*)(a->scratch + second_of(a));
        statistics = to;
        pitch = a->rows;
        for (long long first = 0; first < a->vocab; first += a->piece, ++parts) {
            const long long columns = a->vocab - first < a->piece ? a->vocab - first : a->piece;
            if (int rc = float_logits(a, first, columns, a->scratch, stream)) return rc;
            chained(row_statistics_kernel, (unsigned)a->rows, kThreads, 0, stream, (const float*)a->scratch, pitch_of(a), columns, first, t, to + parts * pitch);
            QMOE_LAUNCH_CHECK("row_statistics_kernel");
        }
    }
    TimedScope timed(KC_HEAD_LOSS, stream);
    chained(join_kernel, (unsigned)ceil_div(a->rows, 32), kThreads, 0, stream, statistics, pitch, parts, t, (float*)a->lse, (float*)a->row_loss);
    QMOE_LAUNCH_CHECK("join_kernel");
    chained(mean_kernel, 1, 1024, 0, stream, (const float*)a->row_loss, t, (float*)a->loss);
    QMOE_LAUNCH_CHECK("mean_kernel");
    return 0;
}

extern "C" int qmoe_pieces_backward(const qmoe_pieces_t* a, uint64_t stream_) {
    if (int rc = pieces_check(a, true)) return rc;
    cudaStream_t stream = (cudaStream_t)stream_;
    const Tables t = tables_of(a);
    const bool bf16 = a->dtype == QMOE_BF16;
    const uint64_t logits = a->scratch, sum = a->scratch + second_of(a);
    const long long pitch = pitch_of(a), parts = parts_of(a);
    const int blocks = ceil_div(pitch, 64), part_blocks = ceil_div(blocks, parts);          // bf16: of the first piece, no other is larger
    const long long out_item = a->weight_gradient == QMOE_BF16 ? 2 : 4;
    for (long long first = 0; first < a->vocab; first += a->piece) {
        const long long columns = a->vocab - first < a->piece ? a->vocab - first : a->piece;
        if (bf16) {
            const PieceGemm g = piece_gemm(a, t, first, columns);
            {
                TimedScope timed(KC_EXPERT_GEMM, stream);
                if (int rc = tc_piece_gradient(g, logits, stream)) return rc;
                if (a->d_hidden)
                    if (int rc = tc_piece_inputs(g, logits, sum, first > 0, part_blocks, stream)) return rc;
            }
            TimedScope timed(KC_WGRAD_GEMM, stream);
            if (a->d_weight)
                if (int rc = tc_piece_weight(g, logits, a->d_weight + first * a->width * out_item, a->weight_gradient == QMOE_BF16, stream)) return rc;
            continue;
        }
        {
            TimedScope timed(KC_EXPERT_GEMM, stream);
            if (int rc = float_logits(a, first, columns, logits, stream)) return rc;
            chained(row_gradient_kernel, (unsigned)a->rows, kThreads, 0, stream, (float*)logits, pitch, columns, first, t, (const float*)a->lse, (const float*)a->gradient);
            QMOE_LAUNCH_CHECK("row_gradient_kernel");
            if (a->d_hidden) {
                SimtGemmArgs g = simt(logits, a->weight + first * a->width * 4, sum, a->rows, a->width, columns);
                g.a_rs = pitch; g.a_cs = 1; g.b_rs = a->width; g.b_cs = 1; g.accumulate = first > 0;
                if (parts > 1) {
                    g.mode = SG_SPLITK; g.k_chunk = (columns + parts - 1) / parts; g.c_slab = a->rows * a->width;
                }
                if (int rc = launch_simt_gemm(g, QMOE_F32, QMOE_F32, QMOE_F32, a->rows, (int)parts, stream)) return rc;
            }
        }
        if (a->d_weight) {
            TimedScope timed(KC_WGRAD_GEMM, stream);
            SimtGemmArgs g = simt(logits, a->inputs, a->d_weight + first * a->width * 4, columns, a->width, a->rows);
            g.a_rs = 1; g.a_cs = pitch; g.b_rs = a->width; g.b_cs = 1;
            if (int rc = launch_simt_gemm(g, QMOE_F32, QMOE_F32, QMOE_F32, columns, 1, stream)) return rc;
        }
    }
    TimedScope timed(KC_OTHER, stream);
    if (a->d_hidden) {
        const unsigned grid = (unsigned)ceil_div(a->rows, kWarps);
        if (bf16)
            chained(scatter_kernel<__nv_bfloat16>, grid, kThreads, 0, stream, (const float*)sum, ceil_div(blocks, part_blocks), bound_of(a->rows) * a->width, t.factor, (const float*)a->gradient, (__nv_bfloat16*)a->d_hidden,
                    t.place, a->rows, a->width);
        else
            chained(scatter_kernel<float>, grid, kThreads, 0, stream, (const float*)sum, (int)parts, a->rows * a->width, nullptr, nullptr, (float*)a->d_hidden, t.place,
                    a->rows, a->width);
        QMOE_LAUNCH_CHECK("scatter_kernel");
    }
    if (a->d_weight && bf16) {
        chained(clear_unwritten_kernel, (unsigned)(2 * sm_count()), kThreads, 0, stream, (uint4*)a->d_weight, a->vocab * a->width * out_item / 16, t.counts);
        QMOE_LAUNCH_CHECK("clear_unwritten_kernel");
    }
    return 0;
}
