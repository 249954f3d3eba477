// Rotation of query and key heads by the angles of each row's position, in one launch, forward and (with the angles' sense reversed, since a
// rotation's transpose is its inverse) backward:
//     (y_a, y_b) = (x_a cos - x_b sin, x_a sin + x_b cos),   angle = p f_i,
// for the pairs (a, b) of a head's first `turned` elements: neighbours (2 i, 2 i + 1), or halves (i, i + turned / 2).  The elements behind are copied.
// The frequencies f_i are the caller's, as 64-bit fractions of a turn: p f_i modulo one turn is an integer product (rotary.cu says why), so that
// scaled frequencies for long contexts are a matter of the host's table alone.
//
// A warp has a row, or a chunk of it where the rows are few, and forms the row's cosines and sines once, a pair to a lane.  The row then goes by in
// units of 16 bytes (halves: two times 16, from both halves), four to a lane in flight.  A unit is read and written by the same lane, so an output may
// lie on its own operand, row on row.
// What bounds it: memory (the L2 where the rows fit it) and, near it, the issue of instructions (45 to 49 % of the cycles), and for few rows the launch.  Forward or backward of
// 8192 rows, 20 heads of 64, bf16: 8 us (42 MB, 5.2 TB/s); 3001 rows, 10 heads of 128 of which 48 elements turn, float32: 6.6 us (31 MB, 4.6 TB/s); 64 rows: 6.5 us with the
// call.  A warp of its own for queries and for keys would form a row's angles twice.
#include "common.cuh"

#include <string.h>

namespace qmoe {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxPairs = 128;
constexpr int kInFlight = 4;
constexpr long long kFarthest = 1ll << 37;

struct RotateParams {
    const void* q;
    const void* k;
    void* q_out;
    void* k_out;
    const int* positions;
    long long offset, q_pitch, k_pitch;
    int rows, time, heads, kv_heads, dim, turned;
    int units, q_units, all_units, chunk;    // 16-byte units (scalar form: elements or pairs) of a head, of a row's queries, of a row, of a warp
    unsigned magic;                          // ceil(2^32 / units): a unit's head
    float sense;
    unsigned long long turns[kMaxPairs];
};

// cosines and sines of the row's pairs, one to a lane, for the whole warp
__device__ __forceinline__ void row_angles(const RotateParams& p, const unsigned long long* turns, float2* angles, int row) {
    const long long position = p.offset + (p.positions ? p.positions[row] : row % p.time);
    for (int i = threadIdx.x & 31; i < p.turned / 2; i += 32) {
        const int part = (int)(((unsigned long long)position * turns[i]) >> 32);             // of 2^32
        float2 v;
        sincospif((float)part * 4.656612873077392578125e-10f, &v.y, &v.x);                   // 2^-31: half turns
        v.y *= p.sense;
        angles[i] = v;
    }
    __syncwarp();
}

template <typename T, bool HALVES>
__global__ void __launch_bounds__(kThreads, HALVES ? 3 : 4)
rotate_kernel(const __grid_constant__ RotateParams p) {
    chain_begin();
    __shared__ __align__(16) float2 s_angles[kWarps][kMaxPairs];
    __shared__ unsigned long long s_turns[kMaxPairs];
    constexpr int V = Vec16<T>::N;
    const int lane = threadIdx.x & 31, row = (int)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int half = p.turned / 2, last = row < p.rows ? min(p.all_units, (int)(blockIdx.y + 1) * p.chunk) : 0;
    const T* q = (const T*)p.q + row * p.q_pitch;
    const T* k = (const T*)p.k + row * p.k_pitch;
    T* q_out = (T*)p.q_out + (long long)row * (p.heads * p.dim);
    T* k_out = (T*)p.k_out + (long long)row * (p.kv_heads * p.dim);
    uint4 a[kInFlight], b[kInFlight];
    // where a unit starts in its row of heads, and where in its head
    auto place = [&](int unit, int& at) {
        const bool query = unit < p.q_units;
        const int mine = query ? unit : unit - p.q_units, head = (int)__umulhi((unsigned)mine, p.magic), in_head = mine - head * p.units;
        at = HALVES && in_head * V >= half ? p.turned + (in_head * V - half) : in_head * V;
        return head * p.dim + at;
    };
    auto fetch = [&](int unit) {
#pragma unroll
        for (int u = 0; u < kInFlight; ++u, unit += 32) {
            if (unit >= last) continue;
            int at;
            const T* from = (unit < p.q_units ? q : k) + place(unit, at);
            a[u] = *reinterpret_cast<const uint4*>(from);
            if (HALVES && at < half) b[u] = *reinterpret_cast<const uint4*>(from + half);
        }
    };
    int unit = (int)blockIdx.y * p.chunk + lane;
    fetch(unit);
    for (int i = threadIdx.x; i < half; i += kThreads) s_turns[i] = p.turns[i];
    __syncthreads();
    if (last == 0) return;
    const float2* angles = s_angles[threadIdx.x >> 5];
    row_angles(p, s_turns, s_angles[threadIdx.x >> 5], row);
    while (true) {
        const int first = unit;
#pragma unroll
        for (int u = 0; u < kInFlight; ++u, unit += 32) {
            if (unit >= last) continue;
            int at;
            T* to = (unit < p.q_units ? q_out : k_out) + place(unit, at);
            float x[V], y[V];
            if (HALVES && at < half) {
                float c[V], d[V];
                Vec16<T>::unpack(a[u], x);
                Vec16<T>::unpack(b[u], y);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float2 r = angles[at + i];
                    c[i] = x[i] * r.x - y[i] * r.y;
                    d[i] = x[i] * r.y + y[i] * r.x;
                }
                *reinterpret_cast<uint4*>(to) = Vec16<T>::pack(c);
                *reinterpret_cast<uint4*>(to + half) = Vec16<T>::pack(d);
            } else if (!HALVES && at < p.turned) {
                Vec16<T>::unpack(a[u], x);
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const float2 r = angles[(at + i) / 2];
                    y[i] = x[i] * r.x - x[i + 1] * r.y;
                    y[i + 1] = x[i] * r.y + x[i + 1] * r.x;
                }
                *reinterpret_cast<uint4*>(to) = Vec16<T>::pack(y);
            } else {
                *reinterpret_cast<uint4*>(to) = a[u];
            }
        }
        if (first - lane + 32 * kInFlight >= last) return;
        fetch(unit);
    }
}

// Any width, pitch and alignment: a pair, or an element behind the turned ones, to a lane.
template <typename T>
__global__ void __launch_bounds__(kThreads)
rotate_scalar_kernel(const __grid_constant__ RotateParams p, int halves) {
    chain_begin();
    __shared__ __align__(16) float2 s_angles[kWarps][kMaxPairs];
    __shared__ unsigned long long s_turns[kMaxPairs];
    const int row = (int)blockIdx.x * kWarps + (threadIdx.x >> 5), half = p.turned / 2;
    for (int i = threadIdx.x; i < half; i += kThreads) s_turns[i] = p.turns[i];
    __syncthreads();
    if (row >= p.rows) return;
    const float2* angles = s_angles[threadIdx.x >> 5];
    row_angles(p, s_turns, s_angles[threadIdx.x >> 5], row);
    const int last = min(p.all_units, (int)(blockIdx.y + 1) * p.chunk);
    for (int unit = (int)blockIdx.y * p.chunk + (threadIdx.x & 31); unit < last; unit += 32) {
        const bool query = unit < p.q_units;
        const int mine = query ? unit : unit - p.q_units, head = mine / p.units, i = mine - head * p.units;
        const T* from = (query ? (const T*)p.q + row * p.q_pitch : (const T*)p.k + row * p.k_pitch) + head * p.dim;
        T* to = (query ? (T*)p.q_out + (long long)row * (p.heads * p.dim) : (T*)p.k_out + (long long)row * (p.kv_heads * p.dim)) + head * p.dim;
        if (i >= half) {
            to[i + half] = from[i + half];
            continue;
        }
        const int first = halves ? i : 2 * i, second = halves ? i + half : 2 * i + 1;
        const float x = Act<T>::load(from + first), y = Act<T>::load(from + second);
        const float2 r = angles[i];
        Act<T>::store(to + first, x * r.x - y * r.y);
        Act<T>::store(to + second, x * r.y + y * r.x);
    }
}

int rotate_check(const qmoe_rotate_t* a) {
    if (!a) return fail_arg("rotate: argument is null");
    if (a->dtype != QMOE_F32 && a->dtype != QMOE_BF16) return fail_arg("rotate: dtype must be QMOE_F32 or QMOE_BF16");
    if (a->batch < 0 || a->time < 0 || a->heads <= 0 || a->kv_heads <= 0) return fail_arg("rotate: sizes must not be negative, head counts positive");
    if (a->dim < 2 || a->dim > 2 * kMaxPairs) return fail_arg("rotate: the head width must lie between 2 and %d", 2 * kMaxPairs);
    if (a->turned < 2 || a->turned > a->dim || a->turned % 2) return fail_arg("rotate: the turned part must be an even number of elements of the head");
    if (a->layout != QMOE_ROTATE_NEIGHBOURS && a->layout != QMOE_ROTATE_HALVES) return fail_arg("rotate: unknown layout");
    // (heads x units^2 below 2^32 keeps the head of a unit exact; the elements of a row in 32 bits)
    if (a->heads > (1 << 16) || a->kv_heads > (1 << 16) || (a->batch && a->time > 0x7fffffff / a->batch)) return fail_arg("rotate: too many rows or heads");
    if (!a->q || !a->k || !a->q_out || !a->k_out || !a->turns) return fail_arg("rotate: null buffer address");
    // (the table's frequencies are off by up to 2^-64 of a turn a position: 2^-27 there, half of what rounding an angle to a float takes)
    if (a->offset <= -kFarthest || a->offset >= kFarthest) return fail_arg("rotate: the offset must lie within 2^37 of 0");
    const uint64_t item = a->dtype == QMOE_BF16 ? 2 : 4;
    if ((a->q | a->k | a->q_out | a->k_out) & (item - 1) || a->positions & 3u || a->turns & 7u) return fail_arg("rotate: misaligned address");
    const uint64_t widths[2] = {(uint64_t)a->heads * a->dim, (uint64_t)a->kv_heads * a->dim}, rows = (uint64_t)a->batch * (uint64_t)a->time;
    if (a->q_pitch < (int64_t)widths[0] || a->k_pitch < (int64_t)widths[1] || a->q_pitch > (1ll << 31) || a->k_pitch > (1ll << 31))
        return fail_arg("rotate: a row pitch must not be below the row's width, nor beyond 2^31");
    // A lane writes where it has read or somewhere else altogether
    struct Span { uint64_t at, bytes; };
    const uint64_t pitches[2] = {(uint64_t)a->q_pitch, (uint64_t)a->k_pitch}, in[2] = {a->q, a->k}, out[2] = {a->q_out, a->k_out};
    auto dense = [&](int i) { return Span{out[i], rows * widths[i] * item}; };
    auto overlap = [](const Span& x, const Span& y) { return x.at < y.at + y.bytes && y.at < x.at + x.bytes; };
    bool apart = !rows || !overlap(dense(0), dense(1));
    for (int i = 0; rows && i < 2; ++i) {
        for (int j = 0; j < 2; ++j) {
            const Span read = {in[j], ((rows - 1) * pitches[j] + widths[j]) * item};
            apart = apart && ((i == j && out[i] == in[j] && pitches[j] == widths[j]) || !overlap(dense(i), read));
        }
        if (a->positions) apart = apart && !overlap(dense(i), Span{a->positions, rows * 4});
    }
    if (!apart) return fail_arg("rotate: an output may lie on its own operand, row on row, and on nothing else");
    return 0;
}

}  // namespace
}  // namespace qmoe

using namespace qmoe;

extern "C" int qmoe_rotate(const qmoe_rotate_t* a, uint64_t stream_) {
    if (int rc = rotate_check(a)) return rc;
    if (!a->batch || !a->time) return 0;
    cudaStream_t stream = (cudaStream_t)stream_;
    TimedScope timed(KC_ELEMENTWISE, stream);
    RotateParams p;
    p.q = (const void*)a->q; p.k = (const void*)a->k; p.q_out = (void*)a->q_out; p.k_out = (void*)a->k_out;
    p.positions = (const int*)a->positions;
    p.offset = a->offset; p.q_pitch = a->q_pitch; p.k_pitch = a->k_pitch;
    p.rows = (int)(a->batch * a->time); p.time = (int)a->time;
    p.heads = a->heads; p.kv_heads = a->kv_heads; p.dim = a->dim; p.turned = a->turned;
    p.sense = a->backward ? -1.f : 1.f;
    memcpy(p.turns, (const void*)a->turns, a->turned / 2 * sizeof(p.turns[0]));
    const int n = a->dtype == QMOE_BF16 ? 8 : 4, half = a->turned / 2;
    const bool halves = a->layout == QMOE_ROTATE_HALVES;
    const int pieces = (halves ? a->dim - half : a->dim) / n;
    const bool vec = a->dim % n == 0 && (halves ? half : a->turned) % n == 0 && a->q_pitch % n == 0 && a->k_pitch % n == 0 && pieces > 1 &&
                     ((a->q | a->k | a->q_out | a->k_out) & 15u) == 0;
    p.units = vec ? pieces : a->dim - half;
    p.magic = vec ? (unsigned)((0x100000000ull + p.units - 1) / p.units) : 0;
    p.q_units = a->heads * p.units;
    p.all_units = (a->heads + a->kv_heads) * p.units;
    // a warp to a row, or several where the rows leave the machine idle, each with at least a pass of its lanes
    const long long most = (p.all_units + 31) / 32, wanted = (long long)sm_count() * 16 / p.rows;
    const int chunks = (int)(wanted < 1 ? 1 : wanted < most ? wanted : most);
    p.chunk = ceil_div(p.all_units, chunks);
    const dim3 grid((unsigned)ceil_div(p.rows, kWarps), (unsigned)ceil_div(p.all_units, p.chunk));
    const bool bf16 = a->dtype == QMOE_BF16;
    if (!vec) {
        if (bf16) chained(rotate_scalar_kernel<__nv_bfloat16>, grid, kThreads, 0, stream, p, (int)halves);
        else chained(rotate_scalar_kernel<float>, grid, kThreads, 0, stream, p, (int)halves);
    } else if (halves) {
        if (bf16) chained(rotate_kernel<__nv_bfloat16, true>, grid, kThreads, 0, stream, p);
        else chained(rotate_kernel<float, true>, grid, kThreads, 0, stream, p);
    } else {
        if (bf16) chained(rotate_kernel<__nv_bfloat16, false>, grid, kThreads, 0, stream, p);
        else chained(rotate_kernel<float, false>, grid, kThreads, 0, stream, p);
    }
    QMOE_LAUNCH_CHECK("rotate_kernel");
    return 0;
}
