// 8-bit paged KV cache: quantised writes (with the heads' norm and rotation in
// the same pass), reads, and causal attention over it. The formats and the
// rules of the stored values are in phonon_gpu.h.
#include <algorithm>

#include "pgpu_common.hpp"
#include "phonon_gpu.h"

namespace pgpu {

// Rows that a call reads or writes once, past the caches.
__device__ inline float4 once_load(const float *p) {
    const f32x4 v = __builtin_nontemporal_load((const f32x4 *)p);
    return make_float4(v.x, v.y, v.z, v.w);
}
__device__ inline void once_store(float *p, float4 v) {
    __builtin_nontemporal_store(f32x4{v.x, v.y, v.z, v.w}, (f32x4 *)p);
}

// One layer of the cache, and the rows of a call (pgpu_kv8, pgpu_kv8_rows).
struct Kv8 {
    int8_t *values;
    float *scales, *open;
    int heads;
    unsigned blocks, slots;
};

struct Kv8Rows {
    const int32_t *tables;
    int table_stride;
    const int32_t *slots, *first, *offsets;
    int rows, max_rows;
};

// Memory that no work-group of a launch writes, at an address that is the same
// for a wave: read through the scalar cache.
template <typename T>
__device__ inline T uniform_load(const T *p) {
    return *(const __attribute__((address_space(4))) T *)p;
}

// A stream's rows, checked: uniform over the work-group.
struct Kv8Span {
    int first, count, row0, slot;
    bool live;
};

// limit: positions must be below it. A stream that breaks a bound is flagged
// (by the thread with `speak`) and left out.
__device__ inline Kv8Span kv8_span(const Kv8 &kv, const Kv8Rows &r, int s, int limit, bool speak,
                                   int *status) {
    Kv8Span x;
    x.first = uniform_load(r.first + s);
    x.slot = uniform_load(r.slots + s);
    x.row0 = r.offsets ? uniform_load(r.offsets + s) : s;
    const int end = r.offsets ? uniform_load(r.offsets + s + 1) : s + 1;
    // 64 bits: any int32 may stand in the arrays.
    const long long count = (long long)end - x.row0;
    const bool wild = x.row0 < 0 || count < 0 || end > r.rows || count > r.max_rows;
    x.count = wild ? 0 : (int)count;
    const long long last = (long long)x.first + x.count;
    const bool bad = wild || (x.first >= 0 && x.count > 0 &&
                              ((unsigned)x.slot >= kv.slots || last > limit ||
                               last > (long long)r.table_stride * kBlockPos));
    x.live = !bad && x.first >= 0 && x.count > 0;
    if (bad && speak) atomicOr(status, 2);
    return x;
}

template <int D>
__device__ inline size_t kv8_tile(const Kv8 &kv, unsigned block, int head) {
    return ((size_t)block * kv.heads + head) * (2 * kBlockPos * D);
}

// Offset of value (position j, dim d) of a block, past its keys: the inverse
// of [j / 4][d % 16][d / 16][j % 4].
template <int D>
__device__ inline int kv8_value_at(int j, int d) {
    return ((j >> 2) * 16 + (d & 15)) * (D / 4) + (d >> 4) * 4 + (j & 3);
}

// max|x| of a block -> its scale. 12 significant bits: see phonon_gpu.h. The
// last clamp keeps 127 s finite.
__device__ inline float kv8_scale(float top) {
    const uint32_t bits = (fbits(top / 127.0f) + 0xFFFu) & ~0xFFFu;
    return fminf(fmaxf(bitsf(bits), 1.17549435e-38f), 0x1.02p+121f);
}

// Byte b of four numbers -> a word; sel = b | (4 + b) << 8.
__device__ inline uint32_t pick4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t sel) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, sel),
                                 __builtin_amdgcn_perm(b, a, sel), 0x05040100u);
}
// LDS between the lanes of one wave: nothing is moved across it.
__device__ inline void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ------------------------------------------------------------------- writing

// A wave holds one (block, head): lane (g, c) has rows 4 g .. 4 g + 3 of the 4
// dims from 4 (c + 16 n) on, n < D / 64: the rows of a byte's word among the
// values, and the dims of one among the keys.
template <int D>
struct Kv8Tile {
    float4 x[D / 64][4];  // [n][row of the four]
};

template <int D>
__device__ inline uint32_t kv8_top(const Kv8Tile<D> &t) {
    uint32_t top = 0;  // |x| orders like its bits: infinities and NaN come out on top
#pragma unroll
    for (int n = 0; n < D / 64; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float4 v = t.x[n][r];
            top = max(max(top, fbits(v.x) & 0x7fffffffu), fbits(v.y) & 0x7fffffffu);
            top = max(max(top, fbits(v.z) & 0x7fffffffu), fbits(v.w) & 0x7fffffffu);
        }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    return top;
}

// The block's 16 rows of keys (p = 0) or values (1) -> the cache. `lds`: 16 D
// bytes of the wave's own. A value that is not finite: a NaN scale, and status
// bit 1. x / s by the reciprocal, which is off by less than 1.6e-5 below 128;
// where that could decide a rounding, by the division.
template <int D>
__device__ inline void kv8_store(const Kv8 &kv, unsigned block, int head, int p,
                                 const Kv8Tile<D> &t, uint32_t *lds, int *status) {
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    int8_t *tile = kv.values + kv8_tile<D>(kv, block, head) + p * kBlockPos * D;
    const uint32_t top = kv8_top<D>(t);
    const bool wild = top >= 0x7f800000u;
    const float s = kv8_scale(bitsf(top)), inverse = 1.0f / s;
#pragma unroll
    for (int n = 0; n < D / 64; n++) {
        float q[4][4], off = 0.0f;  // [row][dim]
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float4 x = t.x[n][r];
            const float f[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const float y = f[d] * inverse;
                q[r][d] = rintf(y);
                off = fmaxf(off, fabsf(y - q[r][d]));
            }
        }
        if (__any(off > 0.5f - 1.6e-5f))
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float4 x = t.x[n][r];
                q[r][0] = rintf(x.x / s);
                q[r][1] = rintf(x.y / s);
                q[r][2] = rintf(x.z / s);
                q[r][3] = rintf(x.w / s);
            }
        uint32_t u[4][4];
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int d = 0; d < 4; d++) u[r][d] = wild ? 0u : (uint32_t)(int)q[r][d];
        // Byte 0 of four numbers -> a word: of a row's dims, or of a dim's rows.
        if (p == 0) {
#pragma unroll
            for (int z = 0; z < 4; z++)
                *(uint32_t *)(tile + (g * 4 + z) * D + n * 64 + c * 4) =
                    pick4(u[z][0], u[z][1], u[z][2], u[z][3], 0x0400u);
        } else {
#pragma unroll
            for (int z = 0; z < 4; z++)
                lds[kv8_value_at<D>(g * 4, n * 64 + c * 4 + z) / 4] =
                    pick4(u[0][z], u[1][z], u[2][z], u[3][z], 0x0400u);
        }
    }
    if (p) {
        wave_lds_fence();
#pragma unroll
        for (int n = 0; n < D / 64; n++)
            *(uint4 *)(tile + (n * 64 + lane) * 16) = ((const uint4 *)lds)[n * 64 + lane];
    }
    if (lane == 0) {
        kv.scales[((size_t)block * kv.heads + head) * 2 + p] = wild ? __builtin_nanf("") : s;
        if (wild) atomicOr(status, 1);
    }
}

struct Kv8Turn {
    const float *qkv;  // rotate: projected rows; else k
    const float *v;
    size_t row_stride;
    int group;
    const float *q_weight, *k_weight;
    float epsilon;
    const float *rope;
    int rope_positions;
    float q_scale;
    float *q_out;
};

// A row's head in the D / 4 dim groups of 16 lanes (D / 64 to a lane):
// normalised (weight), turned, scaled; in 64 bits, rounded once. All 16 lanes
// call it.
template <int D>
__device__ inline void kv8_turn(float4 *x, const float *weight, float epsilon,
                                const float *rope_row, float scale) {
    constexpr int N = D / 64;
    const int c = threadIdx.x & 15;
    double r = 1.0;
    if (weight) {
        double sq = 0.0;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const double a = x[n].x, b = x[n].y, e = x[n].z, f = x[n].w;
            sq += a * a + b * b + e * e + f * f;
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) sq += __shfl_xor(sq, o);
        r = 1.0 / sqrt(sq / D + (double)epsilon);
    }
#pragma unroll
    for (int n = 0; n < N; n++) {
        double y[4] = {x[n].x, x[n].y, x[n].z, x[n].w};
        if (weight) {
            const float4 w = *(const float4 *)(weight + n * 64 + c * 4);
            y[0] = y[0] * r * w.x;
            y[1] = y[1] * r * w.y;
            y[2] = y[2] * r * w.z;
            y[3] = y[3] * r * w.w;
        }
        const float4 cs = *(const float4 *)(rope_row + n * 64 + c * 4);
        const double f = scale;
        x[n] = make_float4((float)((y[0] * cs.x - y[1] * cs.y) * f),
                           (float)((y[0] * cs.y + y[1] * cs.x) * f),
                           (float)((y[2] * cs.z - y[3] * cs.w) * f),
                           (float)((y[2] * cs.w + y[3] * cs.z) * f));
    }
}

__device__ inline bool fine4(float4 x) {
    return isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w);
}

// A wave for each (block of the call's rows, head) of the keys, of the values
// and (rotate) of the queries; no wave waits for another. Bound by HBM: 64 ragged
// prompts of up to 2048 positions, 272 MB of rows in and 68 MB of blocks out, 60 us
// (5.7 TB/s; rows read through the caches 88). With norm and rotation, 16 prompts of
// up to 501, 2 queries a head of 128: 28 us for 115 MB (4.1 TB/s), 40% of the cycles
// in the 64-bit arithmetic.
template <int D, bool ROTATE>
__global__ __launch_bounds__(256, D == 64 ? 6 : 4) void k_kv8_write(Kv8 kv, Kv8Rows rows,
                                                                    Kv8Turn a, int *status) {
    constexpr int N = D / 64;
    __shared__ __align__(16) uint32_t lds[4][D * 4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int s = blockIdx.z, g = lane >> 4, c = lane & 15;
    const Kv8Span span = kv8_span(kv, rows, s,
                                  ROTATE ? a.rope_positions : INT32_MAX - kBlockPos,
                                  threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0, status);
    if (!span.live) return;
    const int end = span.first + span.count;
    const int block = span.first / kBlockPos + (int)blockIdx.y, newest = (end - 1) / kBlockPos;
    const int unit = blockIdx.x * 4 + wave, units = kv.heads * (ROTATE ? 2 + a.group : 2);
    if (block > newest || unit >= units) return;
    bool bad = false;

    if (ROTATE && unit >= 2 * kv.heads) {
        const int head = unit - 2 * kv.heads, width = kv.heads * a.group * D;
        float4 x[4][N];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int p = block * kBlockPos + g * 4 + r;
            const bool in = p >= span.first && p < end;
            const size_t row = (size_t)(span.row0 + (in ? p - span.first : 0));
#pragma unroll
            for (int n = 0; n < N; n++)
                x[r][n] = once_load(a.qkv + row * a.row_stride + head * D + n * 64 + c * 4);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int p = block * kBlockPos + g * 4 + r;
            if (p < span.first || p >= end) continue;  // the same for the row's 16 lanes
            const size_t row = (size_t)(span.row0 + p - span.first);
            kv8_turn<D>(x[r], a.q_weight, a.epsilon, a.rope + (size_t)p * D, a.q_scale);
#pragma unroll
            for (int n = 0; n < N; n++) {
                *(float4 *)(a.q_out + row * width + head * D + n * 64 + c * 4) = x[r][n];
                bad |= !fine4(x[r][n]);
            }
        }
        flag_nonfinite(status, bad);
        return;
    }

    const int head = unit >> 1, part = unit & 1;  // keys, values
    float *slot = kv.open + (((size_t)span.slot * kv.heads + head) * 2 + part) * (kBlockPos * D);
    const float *src = ROTATE ? a.qkv + (size_t)(kv.heads * (a.group + part) + head) * D
                              : (part ? a.v : a.qkv) + (size_t)head * D;
    // Rows of block b: the call's, else what the slot held (only before the
    // call's first row), else 0.
    auto gather = [&](int b, Kv8Tile<D> &t) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int p = b * kBlockPos + g * 4 + r;
            const bool held = p < span.first, in = !held && p < end;
            const float *x = held ? slot + (g * 4 + r) * D
                                  : src + (size_t)(span.row0 + (in ? p - span.first : 0)) * a.row_stride;
#pragma unroll
            for (int n = 0; n < N; n++)
                t.x[n][r] = in || held ? once_load(x + n * 64 + c * 4)
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (ROTATE && part == 0)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int p = b * kBlockPos + g * 4 + r;
                if (p < span.first || p >= end) continue;
                float4 x[N];
#pragma unroll
                for (int n = 0; n < N; n++) x[n] = t.x[n][r];
                kv8_turn<D>(x, a.k_weight, a.epsilon, a.rope + (size_t)p * D, 1.0f);
#pragma unroll
                for (int n = 0; n < N; n++) t.x[n][r] = x[n];
            }
    };
    Kv8Tile<D> t;
    gather(block, t);
    if ((block + 1) * kBlockPos <= end) {
        const int id = uniform_load(rows.tables + (size_t)s * rows.table_stride + block);
        if ((unsigned)id < kv.blocks)
            kv8_store<D>(kv, (unsigned)id, head, part, t, lds[wave], status);
        else if (lane == 0)
            atomicOr(status, 2);
    }
    // The first block's wave, which reads the slot's earlier rows, also replaces
    // them, by the call's rows of the newest block.
    if (blockIdx.y != 0) return;
    if (block != newest) gather(newest, t);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int p = newest * kBlockPos + g * 4 + r;
        if (p < span.first || p >= end) continue;
#pragma unroll
        for (int n = 0; n < N; n++) {
            *(float4 *)(slot + (g * 4 + r) * D + n * 64 + c * 4) = t.x[n][r];
            bad |= !fine4(t.x[n][r]);
        }
    }
    flag_nonfinite(status, bad);
}

// The open slots' full blocks -> the cache, a wave for each (head, keys or values,
// layer, stream).
template <int D>
__global__ __launch_bounds__(256) void k_kv8_close(Kv8 kv, size_t layer_values,
                                                   size_t layer_scales, size_t layer_open,
                                                   const int32_t *tables, int table_stride,
                                                   const int32_t *slots, const int32_t *positions,
                                                   int *status) {
    __shared__ __align__(16) uint32_t lds[4][D * 4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int s = blockIdx.z, layer = blockIdx.y, head = blockIdx.x * 2 + wave / 2, part = wave & 1;
    const int p = uniform_load(positions + s);
    if (p < 0 || p % kBlockPos != kBlockPos - 1 || head >= kv.heads) return;
    const int id = p / kBlockPos < table_stride
                       ? uniform_load(tables + (size_t)s * table_stride + p / kBlockPos) : -1;
    const int slot = uniform_load(slots + s);
    if ((unsigned)id >= kv.blocks || (unsigned)slot >= kv.slots) {
        if (lane == 0) atomicOr(status, 2);
        return;
    }
    kv.values += layer * layer_values;
    kv.scales += layer * layer_scales;
    const float *src = kv.open + layer * layer_open +
                       (((size_t)slot * kv.heads + head) * 2 + part) * (kBlockPos * D);
    Kv8Tile<D> t;
#pragma unroll
    for (int n = 0; n < D / 64; n++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            t.x[n][r] = *(const float4 *)(src + ((lane >> 4) * 4 + r) * D + n * 64 + (lane & 15) * 4);
    kv8_store<D>(kv, (unsigned)id, head, part, t, lds[wave], status);
}

// ------------------------------------------------------------------- reading

// A wave for each (block of the rows read, head). Bound by HBM: 51 us for 68 MB of
// blocks in and 272 MB of rows out (6.7 TB/s).
template <int D>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8 kv, Kv8Rows rows, const int32_t *lengths,
                                                  float *k, float *v, size_t row_stride,
                                                  int *status) {
    constexpr int N = D / 64;
    __shared__ __align__(16) uint32_t lds[4][D * 4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int s = blockIdx.z, head = blockIdx.x * 4 + wave, g = lane >> 4, c = lane & 15;
    const int length = uniform_load(lengths + s);
    const Kv8Span span = kv8_span(kv, rows, s, length,
                                  threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0, status);
    if (!span.live || head >= kv.heads) return;
    const int end = span.first + span.count;
    const int block = span.first / kBlockPos + (int)blockIdx.y;
    if (block * kBlockPos >= end) return;
    float4 x[N][4], y[N][4];
    if (block == (length - 1) / kBlockPos) {
        const float *slot = kv.open + ((size_t)span.slot * kv.heads + head) * (2 * kBlockPos * D);
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int e = (g * 4 + r) * D + n * 64 + c * 4;
                x[n][r] = *(const float4 *)(slot + e);
                y[n][r] = *(const float4 *)(slot + kBlockPos * D + e);
            }
    } else {
        const int id = uniform_load(rows.tables + (size_t)s * rows.table_stride + block);
        if ((unsigned)id >= kv.blocks) {
            if (lane == 0) atomicOr(status, 2);
            return;
        }
        const int8_t *tile = kv.values + kv8_tile<D>(kv, (unsigned)id, head);
        const float2 scale = *(const float2 *)(kv.scales + ((size_t)id * kv.heads + head) * 2);
        uint32_t q[N][4];
#pragma unroll
        for (int n = 0; n < N; n++) {
#pragma unroll
            for (int r = 0; r < 4; r++)
                q[n][r] = *(const uint32_t *)(tile + (g * 4 + r) * D + n * 64 + c * 4);
            ((uint4 *)lds[wave])[n * 64 + lane] =
                *(const uint4 *)(tile + kBlockPos * D + (n * 64 + lane) * 16);
        }
        wave_lds_fence();
#pragma unroll
        for (int n = 0; n < N; n++) {
            uint32_t w[4];  // of dim z: the four rows' bytes
#pragma unroll
            for (int z = 0; z < 4; z++)
                w[z] = lds[wave][kv8_value_at<D>(g * 4, n * 64 + c * 4 + z) / 4];
            auto byte = [](uint32_t a, int i) { return (float)(int8_t)(a >> (8 * i)); };
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[n][r] = make_float4(byte(q[n][r], 0) * scale.x, byte(q[n][r], 1) * scale.x,
                                      byte(q[n][r], 2) * scale.x, byte(q[n][r], 3) * scale.x);
                y[n][r] = make_float4(byte(w[0], r) * scale.y, byte(w[1], r) * scale.y,
                                      byte(w[2], r) * scale.y, byte(w[3], r) * scale.y);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int p = block * kBlockPos + g * 4 + r;
        if (p < span.first || p >= end) continue;
        const size_t at = (size_t)(span.row0 + p - span.first) * row_stride + head * D + c * 4;
#pragma unroll
        for (int n = 0; n < N; n++) {
            once_store(k + at + n * 64, x[n][r]);
            once_store(v + at + n * 64, y[n][r]);
        }
    }
}

// ----------------------------------------------------------------- attention

// The sums are taken on the int8 matrix instruction v_mfma_i32_16x16x64_i8:
// the cache's bytes are its operands as they are stored, nothing is converted.
// A query (and the weights of 64 keys) becomes a fixed-point number of 30 bits
// below its largest element, split into four signed bytes that stand in
// four rows of the other operand: products and sums are exact, and
//   ((b3 * 2^8 + b2) * 2^16 + (b1 * 2^8 + b0)) * step
// is rounded to fp32. An element down to 2^-7 of the largest keeps all its 24
// bits, a smaller one what is above 2^-31 of the largest (three bytes lost 2^-23 of
// it: 2^-9 of dims that lie 2^14 below one of the block's). Four queries fill the 16
// rows (row 4 j + t: byte 3 - t of query j); a lone query stands there four times,
// which costs nothing.

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kNone = -3.0e38f;  // the maximum of no scores

__device__ inline float row16_max(float v) {
    // v_max of the lane 8, 4, 2, 1 apart within each row of 16.
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                     0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, false)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                     0, __builtin_bit_cast(int, v), 0x124, 0xf, 0xf, false)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                     0, __builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, false)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                     0, __builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, false)));
    return v;
}

// Fixed point below `top` (>= 0, the largest magnitude): the power of two that
// takes it above 2^30 / 1.004 and not above 127 * (2^24 + 2^16 + 2^8 + 1), the
// largest sum of four signed bytes (0x11000 carries a significand above 1.992
// into the exponent). Below 2^-96 the step stays at 2^-126.
__device__ inline int fix_exponent(float top) {
    return min(126, 157 - (int)((fbits(top) + 0x11000u) >> 23));
}
__device__ inline float power_of_2(int e) { return bitsf((uint32_t)(127 + e) << 23); }
// The four bytes of the number, each signed: n = sum of byte t * 256^t.
__device__ inline uint32_t fix_bytes(float x, float mul) {
    return ((uint32_t)(int)rintf(x * mul) + 0x80808080u) ^ 0x80808080u;
}
// Which byte of a number stands in row t of its query: the highest in row 0.
__device__ inline uint32_t row_byte(int t) { return 3u - t; }
// At most 128 products of 2^14 to a byte: two bytes' sums together stay below 2^30.
__device__ inline float fix_sum(i32x4 c) {
    return fmaf((float)(c.x * 256 + c.y), 65536.0f, (float)(c.z * 256 + c.w));
}

__device__ inline float lane_value(float v, int lane) {
    return bitsf((uint32_t)__builtin_amdgcn_readlane((int)fbits(v), lane));
}

template <int P>
__device__ inline uint32_t quad_lane(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, P * 0x55, 0xf, 0xf, false);
}

// Bytes of the cache for one row a stream, read once: past the caches, which pays
// where a load instruction takes whole lines (64 streams of up to 2048 keys 16.3 us
// against 19.6, 256 of up to 8187 179 against 202; heads of 128, 48 streams of up to
// 4096 keys 46.6 against 55.5, and 55.9 with half lines and the caches).
__device__ inline i32x4 stream_load16(const int8_t *p) {
    return __builtin_nontemporal_load((const i32x4 *)p);
}

// Lanes 0..3 of 8 get the first half of lane ^ 7 as their second one, and the
// others the second half of lane ^ 7 as their first.
template <int KB>
__device__ inline void trade_halves(i32x4 (&x)[KB]) {
    if constexpr (KB == 2)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int a = x[0][e], b = x[1][e];
            x[0][e] = __builtin_amdgcn_update_dpp(a, b, 0x141, 0xf, 0xa, false);
            x[1][e] = __builtin_amdgcn_update_dpp(b, a, 0x141, 0xf, 0x5, false);
        }
}

struct Kv8Decode {
    const float *q;
    size_t q_stride;
    int group;
    float scale;  // of the scores, times log2 e
    int max_positions, splits, steps;  // a split: steps * W * 64 keys
    // Slot ((s * max_rows + row of the stream) * query heads + head) * splits + split.
    float *part_acc, *part_ml;
    float *out;  // splits = 1: the rows themselves (else NULL)
    size_t out_stride;
};

template <int D, int W, int Q>
struct Kv8DecodeShared {
    __align__(16) uint32_t digits[W][16][16];  // [row][group of lanes, block]
    __align__(16) float own[W][4][16];         // weights of the newest block
    float acc[W][Q][D];
    float m[W][Q], l[W][Q];
};

// One row a stream. A work-group of W waves takes a split's keys of one
// (stream, key head) for Q (1 or 4) of its queries, W * 64 keys a step: a wave's
// 64 are 4 blocks, whose bytes it requests together (8 or 16 KB), the next
// step's as soon as the registers are free: keys after the scores, values
// after their product. Bound by the cache's bytes; no wave waits for another
// before the joint of all W. A step's requests are the same whatever it holds, and
// the last step stands apart, so that the compiler counts what is in flight and a
// step waits for its own bytes only (with branches between them it waited for all:
// 64 streams of 2900 keys, heads of 128 with 4 queries, 62.8 us against 54.8). 256
// streams of up to 8187 keys, heads of 64: 169 us for 1.10 GB, the rate of a plain
// read (6.5 TB/s).
//
// Values: the 16 bytes that a lane (g, i) holds of a block are 4 positions (4 g
// ..) of the dims i, 16 + i, 32 + i and 48 + i. They are an operand as they are
// too: row 4 T + t of the other one has byte t of the weights in word T and
// zeros elsewhere, so that its sums are those of dims 16 T + i.
template <int D, int W, int Q>
__global__ __launch_bounds__(64 * W, D == 64 ? 6 : 4) void k_kv8_decode(Kv8 kv, Kv8Rows rows,
                                                                        Kv8Decode a, int *status) {
    constexpr int KB = D / 64;
    __shared__ Kv8DecodeShared<D, W, Q> sh;
    // Heads vary fastest: with 8 of them a head's passes stay on one XCD (4, 5 or 6
    // heads over as many bytes: 2 to 4% less of them a second, 6.2 TB/s for 6.4).
    const int head = blockIdx.x % kv.heads, j0 = blockIdx.x / kv.heads * Q;
    const int split = blockIdx.y, s = blockIdx.z;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int i = lane & 15, g = lane >> 4;
    int b0 = (split * a.steps * W + wave) * 4;  // the wave's blocks: b0 .. b0 + 3
    const int32_t *table = rows.tables + (size_t)s * rows.table_stride;
    int ids[4];
#pragma unroll
    for (int t = 0; t < 4; t++)
        ids[t] = uniform_load(table + min(b0 + t, rows.table_stride - 1));
    const Kv8Span span = kv8_span(kv, rows, s, a.max_positions,
                                  threadIdx.x == 0 && blockIdx.x == 0 && split == 0, status);
    const int live = min(Q, a.group - j0);  // queries of this work-group
    const int p = span.first;
    if (!span.live) {
        if (a.out && p < 0 && span.count > 0)
            for (int e = threadIdx.x; e < live * D; e += 64 * W)
                a.out[(size_t)s * a.out_stride + ((size_t)head * a.group + j0) * D + e] = 0.0f;
        return;
    }
    if (split * a.steps * W * 64 > p) return;
    const int newest = p / kBlockPos;

    // Where this lane's 16 bytes are: a key's 16 KB from dim 16 KB g on, and the
    // block's values from 16 KB lane on. Two instructions of a wide head each take
    // whole lines: lane and lane ^ 7 have both halves of the one's, then of the
    // other's, and trade.
    int key_at[KB], value_at[KB];
#pragma unroll
    for (int n = 0; n < KB; n++) {
        const int flip = D == 64 || (lane & 7) / 4 == n ? 0 : 7, half = (lane & 7) / 4;
        key_at[n] = (i ^ flip) * D + g * (D / 4) + (D == 64 ? 0 : half * 16);
        value_at[n] = (lane ^ flip) * (D / 4) + (D == 64 ? 0 : half * 16);
    }
    i32x4 kr[4][KB], vr[4][KB];
    float ks[4], vs[4];
    bool wild = false, spoiled = false;
    unsigned on = 0;  // bit t: block t of the step whose keys were requested counts
    // Blocks b .. b + 3; block 0 for one that is not closed or not in the cache, so
    // that every step requests alike and waits for no more than it needs.
    auto load = [&](int b, bool values) {
        if (!values) on = 0;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const bool closed = b + t < newest, in = (unsigned)ids[t] < kv.blocks;
            const unsigned id = closed && in ? (unsigned)ids[t] : 0u;
            if (!values) {
                wild |= closed && !in;
                on |= (closed && in ? 1u : 0u) << t;
            }
            const int8_t *tile = kv.values + kv8_tile<D>(kv, id, head);
            const float *sc = kv.scales + ((size_t)id * kv.heads + head) * 2;
            (values ? vs : ks)[t] = uniform_load(sc + values);
#pragma unroll
            for (int n = 0; n < KB; n++)
                (values ? vr : kr)[t][n] = stream_load16(
                    tile + (values ? kBlockPos * D + value_at[n] : key_at[n]));
        }
    };
    const float *slot = kv.open + ((size_t)span.slot * kv.heads + head) * (2 * kBlockPos * D);

    // Row i of the operand: byte i % 4 of query j0 + i / 4.
    const float *q = a.q + (size_t)s * a.q_stride +
                     ((size_t)head * a.group + min(j0 + (i >> 2), a.group - 1)) * D;
    const uint32_t byte = row_byte(i & 3), sel = byte | (4u + byte) << 8;
    i32x4 qd[KB];
    float step, top = 0.0f;
    auto begin = [&] {
        float4 x[KB][4];
#pragma unroll
        for (int n = 0; n < KB; n++)
#pragma unroll
            for (int k = 0; k < 4; k++)
                x[n][k] = *(const float4 *)(q + g * (D / 4) + n * 16 + k * 4);
        // The order of the requests is the order in which they are waited for.
        __builtin_amdgcn_sched_barrier(0);
        load(b0, false);
        __builtin_amdgcn_sched_barrier(0);
        load(b0, true);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < KB; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float4 v = x[n][k];
                top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)),
                                       fmaxf(fabsf(v.z), fabsf(v.w))));
            }
        top = xor16_32_max(top);
        const int e = fix_exponent(top);
        const float mul = power_of_2(e);
#pragma unroll
        for (int n = 0; n < KB; n++)
#pragma unroll
            for (int k = 0; k < 4; k++)
                qd[n][k] = (int)pick4(fix_bytes(x[n][k].x, mul), fix_bytes(x[n][k].y, mul),
                                      fix_bytes(x[n][k].z, mul), fix_bytes(x[n][k].w, mul), sel);
        // From here on this lane's query is j0 + g (rows 4 g .. 4 g + 3). Fixed point
        // cannot say that it is infinite.
        step = __shfl(top < INFINITY ? a.scale * power_of_2(-e) : __builtin_nanf(""), g * 4);
    };
    // This lane's query is j0 + g in m and l; acc: dims lane, 64 + lane of each.
    float m = kNone, l = 0.0f, acc[Q][KB];
#pragma unroll
    for (int j = 0; j < Q; j++)
#pragma unroll
        for (int k = 0; k < KB; k++) acc[j][k] = 0.0f;

    auto attend = [&](bool more) {
        const unsigned count = on;
        if (more)
#pragma unroll
            for (int t = 0; t < 4; t++)
                ids[t] = uniform_load(table + min(b0 + 4 * W + t, rows.table_stride - 1));
        // Scores, in units of log 2: lane (g, i) key i of each block.
        float w[4], mx = m;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            i32x4 c = {0, 0, 0, 0};
            trade_halves<KB>(kr[t]);
#pragma unroll
            for (int k = 0; k < KB; k++)
                c = __builtin_amdgcn_mfma_i32_16x16x64_i8(qd[k], kr[t][k], c, 0, 0, 0);
            w[t] = count >> t & 1 ? fix_sum(c) * (step * ks[t]) : -INFINITY;
            mx = fmaxf(mx, w[t]);
        }
        if (more) load(b0 + 4 * W, false);
        mx = row16_max(mx);
        const float shrink = __builtin_amdgcn_exp2f(m - mx);  // m = kNone: 0
        m = mx;
        float sum = 0.0f, big = 0.0f;
        // The weights times their blocks' value scales, in fixed point below
        // the largest of the query's 64; byte t of four keys in a row's word.
#pragma unroll
        for (int t = 0; t < 4; t++) {
            w[t] = __builtin_amdgcn_exp2f(w[t] - m);
            sum += w[t];
            const float v = count >> t & 1 ? vs[t] : 0.0f;
            // A block whose values were not finite: fixed point cannot say so.
            spoiled |= v != v;
            w[t] *= v;
            big = fmaxf(big, w[t]);
        }
        l = fmaf(l, shrink, row16_sum(sum));
        const int f = fix_exponent(row16_max(big));
        const float mul = power_of_2(f), back = power_of_2(-f);
        i32x4 word;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const uint32_t u = fix_bytes(w[t], mul);
            word[t] = (int)pick4(quad_lane<0>(u), quad_lane<1>(u), quad_lane<2>(u),
                                 quad_lane<3>(u), sel);
        }
        *(i32x4 *)&sh.digits[wave][g * 4 + (i & 3)][(i >> 2) * 4] = word;
        wave_lds_fence();
#pragma unroll
        for (int t = 0; t < 4; t++) trade_halves<KB>(vr[t]);
#pragma unroll
        for (int j = 0; j < Q; j++) {
            const i32x4 pd = *(const i32x4 *)&sh.digits[wave][j * 4 + (i & 3)][g * 4];
            i32x4 c[KB];
#pragma unroll
            for (int k = 0; k < KB; k++) c[k] = i32x4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int x = pd[t], z = i >> 2;
                const i32x4 row = {z == 0 ? x : 0, z == 1 ? x : 0, z == 2 ? x : 0, z == 3 ? x : 0};
#pragma unroll
                for (int k = 0; k < KB; k++)
                    c[k] = __builtin_amdgcn_mfma_i32_16x16x64_i8(row, vr[t][k], c[k], 0, 0, 0);
            }
            const float one = Q == 1 ? back : lane_value(back, j * 16);
            const float less = Q == 1 ? shrink : lane_value(shrink, j * 16);
#pragma unroll
            for (int k = 0; k < KB; k++) acc[j][k] = fmaf(fix_sum(c[k]), one, acc[j][k] * less);
        }
        b0 += 4 * W;
        if (more) load(b0, true);
        wave_lds_fence();
    };
    // The last step apart: no branch stands between a request and its wait. A wave
    // without a step requests nothing, where that comes often enough to be worth
    // the branch: contexts of 16 keys 4.2 us alone for 5.4, 64 streams of up to 300 6.3
    // for 7.5, of up to 1500 14.1 for 13.8; dealt, 48 of 4096 with 4 queries 42 for 41.
    int steps = b0 < newest ? min(a.steps, (newest - b0 - 1) / (4 * W) + 1) : 0;
    if (W == 4 || steps > 0) {
        begin();
        // Not known to be above 0: the two ways out of the loop would then be given
        // registers of their own, and spill.
        if (W > 4) asm("" : "+s"(steps));
        for (; steps > 1; steps--) attend(true);
        if (steps > 0) attend(false);
    }
    // The newest block, in fp32: by the wave after the one whose blocks end there,
    // which has had a step less.
    if (newest / (a.steps * W * 4) == split && (newest / 4 + 1) % W == wave) {
        f32x4 c = {0.f, 0.f, 0.f, 0.f};
        // The values are requested with the keys (64 streams of up to 2048 keys 15.6
        // us, 16.3 with a row at a time after the weights).
        float own[kBlockPos][KB];
#pragma unroll
        for (int n = 0; n < kBlockPos; n++)
#pragma unroll
            for (int k = 0; k < KB; k++)
                own[n][k] = slot[kBlockPos * D + n * D + k * 64 + lane];
#pragma unroll
        for (int k = 0; k < KB * 4; k++) {
            const int d = k / 4 * 64 + g * 16 + k % 4 * 4;
            const float4 y = *(const float4 *)(slot + i * D + d);
            float4 v = *(const float4 *)(q + d);
            if (W > 4)
                top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)),
                                       fmaxf(fabsf(v.z), fabsf(v.w))));
            if (i & 3) v = make_float4(0.f, 0.f, 0.f, 0.f);
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(v.x, y.x, c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(v.y, y.y, c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(v.z, y.z, c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(v.w, y.w, c, 0, 0, 0);
        }
        float w = newest * kBlockPos + i <= p ? c.x * a.scale : -INFINITY;
        // An infinite query's scores may all be -inf.
        if (__any(!(top < INFINITY)) && !(__shfl(xor16_32_max(top), g * 4) < INFINITY))
            w = __builtin_nanf("");
        const float mx = row16_max(fmaxf(m, w)), shrink = __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        w = __builtin_amdgcn_exp2f(w - m);
        l = fmaf(l, shrink, row16_sum(w));
        sh.own[wave][g][i] = w;
        wave_lds_fence();
        // Rows past the position may hold anything: left out.
#pragma unroll
        for (int j = 0; j < Q; j++) {
            const float less = Q == 1 ? shrink : lane_value(shrink, j * 16);
#pragma unroll
            for (int k = 0; k < KB; k++) acc[j][k] *= less;
        }
#pragma unroll
        for (int n = 0; n < kBlockPos; n++)
            if (newest * kBlockPos + n <= p)
#pragma unroll
                for (int k = 0; k < KB; k++) {
#pragma unroll
                    for (int j = 0; j < Q; j++)
                        acc[j][k] = fmaf(sh.own[wave][j][n], own[n][k], acc[j][k]);
                }
    }
    if (wild && lane == 0) atomicOr(status, 2);
    if (spoiled) l = __builtin_nanf("");
#pragma unroll
    for (int j = 0; j < Q; j++)
#pragma unroll
        for (int k = 0; k < KB; k++) sh.acc[wave][j][k * 64 + lane] = acc[j][k];
    if (g < Q && i == 0) {
        sh.m[wave][g] = m;
        sh.l[wave][g] = l;
    }
    bool bad = !(top < INFINITY);
    __syncthreads();
    for (int e = threadIdx.x; e < live * D; e += 64 * W) {
        const int j = e / D, d = e % D;
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < W; n++) mx = fmaxf(mx, sh.m[n][j]);
        float total = 0.0f, o = 0.0f;
#pragma unroll
        for (int n = 0; n < W; n++) {
            // A wave past the context: l = 0, m = kNone, acc = 0.
            const float c = __builtin_amdgcn_exp2f(sh.m[n][j] - mx);
            total = fmaf(sh.l[n][j], c, total);
            o = fmaf(sh.acc[n][j][d], c, o);
        }
        const size_t qh = (size_t)head * a.group + j0 + j;
        if (a.out) {
            o = o / total;
            a.out[(size_t)s * a.out_stride + qh * D + d] = o;
            bad |= !isfinite(o);
        } else {
            const size_t at = ((size_t)s * kv.heads * a.group + qh) * a.splits + split;
            a.part_acc[at * D + d] = o;
            if (d == 0) *(float2 *)(a.part_ml + at * 2) = make_float2(mx, total);
        }
    }
    flag_nonfinite(status, bad);
}

// Runs of rows: a work-group of 4 waves takes 4 tiles of 16 rows of one query
// head each (the query heads of a key head side by side), and passes over the
// keys 64 at a time: each wave turns one block's bytes into fp16 (exact) in
// LDS, where all four read them, while the next 64 keys' bytes are on their
// way. Scores are taken keys by rows (K Q^T), so that a lane holds 16 of its
// row's scores and the weights are the next product's operand as they stand
// (O^T = V^T P^T). A query and a weight are two fp16 terms (22 bits), each
// product with the cache's whole numbers exact in fp32. The running maximum is
// a whole number (in units of log 2), so that rescaling is exact and rare. The
// weights carry their block's value scale times 2^lift, which keeps them below
// 2^15 and their low terms normal: with every scale so far within 2^4 of the first
// block's, one lift for all rows; else each row's own, from the largest weight
// times scale among the keys that it sees (so no row loses bits to a block that it
// does not see or hardly weighs; 8187 rows 227 us where scales are 2^6 apart, 187 in
// the same run where they are alike).
// Bound by vector instructions: a run of 8187 rows over 8 heads of 64 takes 167 us (183
// on another card; 0.41 PFLOP/s of the formula's, 0.82 with the terms'), 249 instructions
// a tile and chunk in 69% of the cycles, the matrix cores busy in 32%. Tiles of 16 rows
// keep 4 waves a SIMD (two tiles a wave, half the waves: 244); a work-group of 8 waves,
// which would share the conversion by twice the rows, waits at its barriers (192). Short
// runs are bound by the chain within a chunk, 1.1 to 1.5 us.
struct Kv8Run {
    const float *q;
    size_t q_stride;
    int group;
    float scale;  // of the scores, times log2 e
    int max_positions, splits;
    float *part_acc, *part_ml;
    float *out;  // splits = 1: the rows themselves
    size_t out_stride;
};

template <int D>
struct Kv8RunShared {
    f16x8 k[2][4][D / 32][64];      // [buffer][block][step][lane]
    f16x8 v[2][2][D / 16][64];      // [buffer][pair of blocks][16 dims][lane]
    float2 scale[2][4];
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// Four signed bytes -> fp16: 0x6400 | (byte ^ 0x80) is 1152 + byte.
__device__ inline f16x4 bytes_f16(int x) {
    const uint32_t u = (uint32_t)x ^ 0x80808080u;
    const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const uint32_t low = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    const uint32_t high = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    const f16x2 a = __builtin_bit_cast(f16x2, low) + off;
    const f16x2 b = __builtin_bit_cast(f16x2, high) + off;
    return f16x4{a.x, a.y, b.x, b.y};
}

// x, y -> two fp16 terms, both truncated: hi + lo has 22 bits of them. The
// remainder is one v_fma_mix_f32, which reads an fp16 half as it stands.
__device__ inline void split_pair(float x, float y, f16x2 &hi, f16x2 &lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
    const uint32_t u = __builtin_bit_cast(uint32_t, h);
    float rx, ry;
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rx) : "v"(u), "v"(x));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(ry) : "v"(u), "v"(y));
    hi = __builtin_bit_cast(f16x2, h);
    lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(rx, ry));
}

// Pairs of terms -> an operand of 8.
__device__ inline f16x8 join_pairs(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    const i32x4 x = {__builtin_bit_cast(int, a), __builtin_bit_cast(int, b),
                     __builtin_bit_cast(int, c), __builtin_bit_cast(int, d)};
    return __builtin_bit_cast(f16x8, x);
}

// The largest of three; NaN does not count.
__device__ inline float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// The largest over lanes 16 and 32 apart, without the quieting of NaN that fmaxf adds
// to each operand (8187 rows 164.9 us, 166.8 with it).
__device__ inline float quarters_max(float v) {
    auto x = __builtin_amdgcn_permlane16_swap(fbits(v), fbits(v), false, false);
    v = max3(__builtin_bit_cast(float, (uint32_t)x[0]), __builtin_bit_cast(float, (uint32_t)x[1]),
             __builtin_bit_cast(float, (uint32_t)x[1]));
    x = __builtin_amdgcn_permlane32_swap(fbits(v), fbits(v), false, false);
    return max3(__builtin_bit_cast(float, (uint32_t)x[0]), __builtin_bit_cast(float, (uint32_t)x[1]),
                __builtin_bit_cast(float, (uint32_t)x[1]));
}

template <int D>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void k_kv8_run(Kv8 kv, Kv8Rows rows, Kv8Run a,
                                                                  int *status) {
    constexpr int KB = D / 64, KS = D / 32, T = D / 16;
    __shared__ Kv8RunShared<D> sh;
    // Heads fastest (with 8 of them a head's keys stay in one XCD's L2), the
    // longest rows first, and every second 256 work-groups the other way round: a
    // CU, which gets each 256th, has long and short ones.
    const int s = blockIdx.z, head = blockIdx.x % kv.heads, split = blockIdx.x / kv.heads;
    const int plane = gridDim.x * gridDim.y;
    int bx = gridDim.y - 1 - blockIdx.y;
    if (plane <= 256) {
        if ((int)((size_t)blockIdx.z * plane / 256) & 1) bx = blockIdx.y;
    } else {
        const int turn = max(1, 256 / (int)gridDim.x), lap = blockIdx.y / turn;
        if (lap & 1)
            bx = gridDim.y - min((lap + 1) * turn, (int)gridDim.y) + (blockIdx.y - lap * turn);
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int i = lane & 15, g = lane >> 4;
    const Kv8Span span = kv8_span(kv, rows, s, a.max_positions,
                                  threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0, status);
    const int tiles = (span.count + 15) / 16 * a.group;
    if (bx * 4 >= tiles) return;
    const int tile = bx * 4 + wave, r0 = tile / a.group * 16;
    const int qh = head * a.group + tile % a.group;
    const int live = tile < tiles ? min(16, span.count - r0) : 0;  // rows of this wave
    const size_t row = (size_t)(span.row0 + (live > 0 ? r0 + min(i, live - 1) : 0));
    if (!span.live) {
        if (span.first < 0 && split == 0 && i < live) {
            float *dst = a.out + row * a.out_stride + (size_t)qh * D;
            for (int t = 0; t < T; t++)
                *(float4 *)(dst + t * 16 + g * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        return;
    }
    const int end = span.first + span.count, newest = (end - 1) / kBlockPos;
    const int top = span.first + min(span.count, (min(bx * 4 + 3, tiles - 1) / a.group + 1) * 16) - 1;
    const int keys = min(newest * kBlockPos, top + 1);  // of blocks, to be seen by some row here
    // Splits take the chunks in turn, so that each has its share of every row's keys.
    const int c0 = split, stride = a.splits, c1 = (keys + 63) / 64;
    const int p0 = span.first + r0, p = i < live ? p0 + i : -1;  // this lane's row
    const int wave_top = p0 + live - 1;
    const float *slot = kv.open + ((size_t)span.slot * kv.heads + head) * (2 * kBlockPos * D);

    // The wave's queries, two terms, scaled to a largest element in [2^14, 2^15).
    const float *q = a.q + row * a.q_stride + (size_t)qh * D;
    f16x8 qhi[KS], qlo[KS];
    float qs, biggest = 0.0f;
    {
        float4 x[KB][4];
#pragma unroll
        for (int n = 0; n < KB; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float4 v = *(const float4 *)(q + n * 64 + g * 16 + k * 4);
                x[n][k] = v;
                biggest = fmaxf(biggest, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)),
                                               fmaxf(fabsf(v.z), fabsf(v.w))));
            }
        biggest = xor16_32_max(biggest);
        const int e = min(126, 141 - (int)(fbits(biggest) >> 23));
        // The factor of the scores stays above 0, for a scale of 0 too.
        const float mul = a.scale == 0.0f ? 0.0f : copysignf(power_of_2(e), a.scale);
        qs = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * power_of_2(-e);
#pragma unroll
        for (int n = 0; n < KB; n++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                f16x2 h[4], o[4];
#pragma unroll
                for (int z = 0; z < 2; z++) {
                    const float4 v = x[n][k * 2 + z];
                    split_pair(v.x * mul, v.y * mul, h[z * 2], o[z * 2]);
                    split_pair(v.z * mul, v.w * mul, h[z * 2 + 1], o[z * 2 + 1]);
                }
                qhi[n * 2 + k] = join_pairs(h[0], h[1], h[2], h[3]);
                qlo[n * 2 + k] = join_pairs(o[0], o[1], o[2], o[3]);
            }
    }

    // Chunk c: its bytes requested, then turned into LDS; wave w takes block w.
    // The block's id and scales of the j-th chunk wait in lane j (j below 64, then
    // the next 64): no chunk waits for its own.
    i32x4 kr[KB], vr[KB];
    int id_of = 0;
    float2 scale_of = make_float2(1.0f, 0.0f), sc;
    bool wild = false;
    const int32_t *table = rows.tables + (size_t)s * rows.table_stride;
    constexpr int kNear = 4;
    auto exponent = [](float x) { return (int)(fbits(x) >> 23 & 255u) - 127; };
    int usual = 0;  // the value scale's of this work-group's first block
    auto look_up = [&](int c) {
        const int at = c + lane * stride, b = at * 4 + wave;
        const bool in = at < c1 && b * kBlockPos < keys;
        const int raw = in ? table[b] : 0, front = table[c0 * 4];
        wild |= (unsigned)raw >= kv.blocks;
        id_of = (unsigned)raw < kv.blocks ? raw : 0;
        usual = exponent(kv.scales[((size_t)((unsigned)front < kv.blocks ? front : 0) * kv.heads +
                                    head) * 2 + 1]);
        scale_of = make_float2(1.0f, 0.0f);
        if (in) {
            scale_of = *(const float2 *)(kv.scales + ((size_t)id_of * kv.heads + head) * 2);
            // A block whose values were not finite: its scores say so instead, to
            // the rows that see it.
            if (scale_of.y != scale_of.y) scale_of = make_float2(scale_of.y, 0.0f);
            // The sign says that it is far from the first block's.
            if (scale_of.y != 0.0f && abs(exponent(scale_of.y) - usual) > kNear)
                scale_of.y = -scale_of.y;
            // A block that is not in the cache is left out: its scores, which are NaN
            // to the maximum, become -inf.
            if ((unsigned)raw >= kv.blocks) scale_of = make_float2(__builtin_nanf(""), -0.0f);
        }
    };
    auto request = [&](int c, int nth) {
        const int j = nth & 63;
        if (j == 0) look_up(c);
        const unsigned id = (unsigned)__builtin_amdgcn_readlane(id_of, j);
        sc = make_float2(lane_value(scale_of.x, j), lane_value(scale_of.y, j));
        // Past the keys: block 0's bytes, whose keys are hidden and whose scale is 0.
        const int8_t *tl = kv.values + kv8_tile<D>(kv, id, head);
#pragma unroll
        for (int n = 0; n < KB; n++) {
            kr[n] = *(const i32x4 *)(tl + i * D + n * 64 + g * 16);
            vr[n] = *(const i32x4 *)(tl + kBlockPos * D + lane * (D / 4) + n * 16);
        }
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int n = 0; n < KB; n++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const f16x4 x = bytes_f16(kr[n][k * 2]), y = bytes_f16(kr[n][k * 2 + 1]);
                sh.k[buf][wave][n * 2 + k][lane] =
                    __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
        for (int t = 0; t < T; t++)
            *((f16x4 *)&sh.v[buf][wave >> 1][t][lane] + (wave & 1)) = bytes_f16(vr[t / 4][t % 4]);
        if (lane == 0) sh.scale[buf][wave] = sc;
    };

    float m = kNone, l = 0.0f;  // l: of this lane's keys
    f32x4 acc[T];
#pragma unroll
    for (int t = 0; t < T; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // acc holds the values' sums times 2^lift. A scale within 2^kNear: below 2^15.
    int lift = 0;
    bool apart = false;  // a scale so far was not

    auto attend = [&](int buf, int c, bool masked) {
        float2 bs[4];
#pragma unroll
        for (int t = 0; t < 4; t++) bs[t] = sh.scale[buf][t];
        f32x4 w[4];
        // The last key that this lane's row sees, from its own first one on.
        const int last = min(p, keys - 1) - c * 64 - g * 4;
#pragma unroll
        for (int t = 0; t < 4; t++) w[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; k++) {
            f16x8 kk[4];
#pragma unroll
            for (int t = 0; t < 4; t++) kk[t] = sh.k[buf][t][k][lane];
#pragma unroll
            for (int t = 0; t < 4; t++)
                w[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[t], qhi[k], w[t], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < 4; t++)
                w[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[t], qlo[k], w[t], 0, 0, 0);
        }
        if (masked)
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (t * 16 + r > last) w[t][r] = -INFINITY;
        float f[4], mx = kNone;
#pragma unroll
        for (int t = 0; t < 4; t += 2) {
            // A factor is not negative; NaN (a block that was not finite, or a
            // factor that fell to 0 times a hidden key) does not count.
            f[t] = bs[t].x * qs, f[t + 1] = bs[t + 1].x * qs;
            mx = max3(mx, max3(max3(w[t][0], w[t][1], w[t][2]), w[t][3], w[t][3]) * f[t],
                      max3(max3(w[t + 1][0], w[t + 1][1], w[t + 1][2]), w[t + 1][3],
                           w[t + 1][3]) * f[t + 1]);
        }
        // A whole number; not below the last one.
        const float least = ceilf(quarters_max(mx)), mn = max3(m, least, least);
        uint32_t signs = 0;
#pragma unroll
        for (int t = 0; t < 4; t++) signs |= fbits(bs[t].y);
        apart |= (int)__builtin_amdgcn_readfirstlane(signs) < 0;
        if (apart || __any(mn != m)) {
            const float shrink = __builtin_amdgcn_exp2f(m - mn);
            l *= shrink;
            float both = shrink;
            if (apart) {
                // The exponent that no weight times scale of this row passes; and not so
                // far below a scale that it sees that 2^lift times that overflows.
                float large = kNone, seen = kNone;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const float e = (float)(exponent(bs[t].y) + 1);
                    const float best = max3(max3(w[t][0], w[t][1], w[t][2]), w[t][3], w[t][3]);
                    large = max3(large, fmaf(best, f[t], e), large);
                    if (!masked || t * 16 <= last) seen = fmaxf(seen, e);
                    if (fbits(bs[t].y) == 0x80000000u) {  // no block
                        w[t] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                        f[t] = 1.0f;
                    }
                }
                large = ceilf(quarters_max(large)) - mn;
                const float next = fminf(fminf((float)lift + (mn - m), 14.0f - large),
                                         100.0f - quarters_max(seen));
                both = __builtin_amdgcn_exp2f((m - mn) + (next - (float)lift));
                lift = (int)next;
            }
#pragma unroll
            for (int t = 0; t < T; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[t][r] *= both;
            m = mn;
        }
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                w[t][r] = __builtin_amdgcn_exp2f(fmaf(w[t][r], f[t], -m));
        if (masked)
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (t * 16 + r > last) w[t][r] = 0.0f;
        f16x2 hi[4][2], lo[4][2];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const float z = ldexpf(fabsf(bs[t].y), lift);
#pragma unroll
            for (int r = 0; r < 4; r++) l += w[t][r];
            split_pair(w[t][0] * z, w[t][1] * z, hi[t][0], lo[t][0]);
            split_pair(w[t][2] * z, w[t][3] * z, hi[t][1], lo[t][1]);
        }
        const f16x8 ph[2] = {join_pairs(hi[0][0], hi[0][1], hi[1][0], hi[1][1]),
                             join_pairs(hi[2][0], hi[2][1], hi[3][0], hi[3][1])};
        const f16x8 pl[2] = {join_pairs(lo[0][0], lo[0][1], lo[1][0], lo[1][1]),
                             join_pairs(lo[2][0], lo[2][1], lo[3][0], lo[3][1])};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int t0 = 0; t0 < T; t0 += 4) {
                f16x8 v[4];
#pragma unroll
                for (int t = 0; t < 4; t++) v[t] = sh.v[buf][n][t0 + t][lane];
#pragma unroll
                for (int t = 0; t < 4; t++)
                    acc[t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[t], ph[n],
                                                                         acc[t0 + t], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < 4; t++)
                    acc[t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[t], pl[n],
                                                                         acc[t0 + t], 0, 0, 0);
            }
    };

    if (c0 < c1) {
        request(c0, 0);
        lift = 14 - usual - kNear;
        stage(0);
        __syncthreads();
        for (int c = c0, n = 0; c < c1; c += stride, n++) {
            const int buf = n & 1;
            const bool more = c + stride < c1;
            if (more) request(c + stride, n + 1);
            if (live > 0 && c * 64 <= wave_top)
                attend(buf, c, c * 64 + 63 > p0 || c * 64 + 64 > keys || live < 16);
            if (more) stage(buf ^ 1);
            __syncthreads();
        }
    }
    if (__any(wild) && lane == 0) atomicOr(status, 2);
    if (live == 0) return;

    // The newest block, in fp32 on the fp32 matrix instruction.
#pragma unroll
    for (int t = 0; t < T; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) acc[t][r] = ldexpf(acc[t][r], -lift);
    if (split == newest / 4 % stride && wave_top >= newest * kBlockPos) {
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < KB; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float4 y = *(const float4 *)(slot + i * D + n * 64 + g * 16 + k * 4);
                const float4 z = *(const float4 *)(q + n * 64 + g * 16 + k * 4);
                x = __builtin_amdgcn_mfma_f32_16x16x4f32(y.x, z.x, x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_16x16x4f32(y.y, z.y, x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_16x16x4f32(y.z, z.z, x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_16x16x4f32(y.w, z.w, x, 0, 0, 0);
            }
        // Values [key 4 g + r][16 t + i]; rows past the last may hold anything.
        // A value that is not finite makes its key's weight NaN for the rows that
        // see it, and is left out of the product, where it would reach all rows.
        float v[T][4];
        uint32_t odd = 0;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const bool in = newest * kBlockPos + g * 4 + r < end;
#pragma unroll
            for (int t = 0; t < T; t++) {
                const float y = slot[kBlockPos * D + (g * 4 + r) * D + t * 16 + i];
                const bool fine = isfinite(y);
                v[t][r] = in && fine ? y : 0.0f;
                if (in && !fine) odd |= 1u << r;
            }
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) odd |= (uint32_t)__shfl_xor((int)odd, o);
        float mx = kNone;
        f32x4 w;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            w[r] = newest * kBlockPos + g * 4 + r <= p ? x[r] * a.scale : -INFINITY;
            mx = fmaxf(mx, w[r]);
        }
        mx = xor16_32_max(mx);
        // The last maximum as it is: a row of one key gets that key's value.
        const float mn = fmaxf(m, mx), shrink = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= shrink;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const bool seen = w[r] != -INFINITY;
            w[r] = seen ? __builtin_amdgcn_exp2f(w[r] - m) : 0.0f;
            if (seen && (odd >> r & 1)) w[r] = __builtin_nanf("");
            l += w[r];
        }
#pragma unroll
        for (int t = 0; t < T; t++) {
#pragma unroll
            for (int r = 0; r < 4; r++) acc[t][r] *= shrink;
#pragma unroll
            for (int r = 0; r < 4; r++)
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[t][r], w[r], acc[t], 0, 0, 0);
        }
    }
    l = xor16_32_sum(l);
    bool bad = false;
    if (i < live) {
        const size_t at = (((size_t)s * rows.max_rows + r0 + i) * kv.heads * a.group + qh) *
                              a.splits + split;
        float *dst = a.splits == 1 ? a.out + row * a.out_stride + (size_t)qh * D : a.part_acc + at * D;
        // A sum of 0 over keys that the row sees: their blocks were left out, which
        // gives zeros, or all scores are -inf, which does not come out finite.
        if (l == 0.0f && p >= c0 * 64) {
            bool lost = false;
            for (int b = 0; b < newest && b * kBlockPos <= p; b++)
                lost |= (unsigned)table[b] >= kv.blocks;
            if (!lost) l = __builtin_nanf("");
        }
        const float f = a.splits > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int t = 0; t < T; t++) {
            const float4 o = make_float4(acc[t][0] * f, acc[t][1] * f, acc[t][2] * f, acc[t][3] * f);
            bad |= !(isfinite(o.x) && isfinite(o.y) && isfinite(o.z) && isfinite(o.w));
            *(float4 *)(dst + t * 16 + g * 4) = o;
        }
        if (a.splits > 1 && g == 0) *(float2 *)(a.part_ml + at * 2) = make_float2(m, l);
        bad |= !(biggest < INFINITY);
    }
    flag_nonfinite(status, bad);
}

// The splits of a row's query head joined: D / 4 lanes for 4 dims each, times G
// that share the splits. `keys`: of a split, or 0: every split has keys of every
// row, or says that it has none. Eight splits' parts are on their way at once. Bound
// by two dependent loads and the launch: 4 to 5 us beside 2 to 11 splits.
template <int D, int G>
__global__ __launch_bounds__(256) void k_kv8_join(Kv8 kv, Kv8Rows rows, const float *part_acc,
                                                  const float *part_ml, int group,
                                                  int max_positions, int splits, int keys,
                                                  float *out, size_t out_stride, int *status) {
    constexpr int L = D / 4, M = L * G;
    const int s = blockIdx.z, wide = kv.heads * group;
    const size_t e = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int lane = (int)(e % M), share = lane / L, d = lane % L * 4;
    const int qh = (int)(e / M % wide);
    const size_t i = e / M / wide;
    const Kv8Span span = kv8_span(kv, rows, s, max_positions, false, status);
    if (i >= (size_t)span.count || (!span.live && span.first >= 0)) return;
    const size_t row = span.row0 + i;
    float *dst = out + row * out_stride + (size_t)qh * D + d;
    if (!span.live) {
        if (share == 0) *(float4 *)dst = make_float4(0.f, 0.f, 0.f, 0.f);
        return;
    }
    const int n = keys ? (span.first + (int)i) / keys + 1 : splits;
    const size_t at = (((size_t)s * rows.max_rows + i) * wide + qh) * splits;
    // Lane j of the M has split j's maximum and sum, and the next M's.
    float mx = -INFINITY, total = 0.0f;
    for (int j = lane; j < n; j += M) mx = fmaxf(mx, part_ml[(at + j) * 2]);
#pragma unroll
    for (int z = 1; z < M; z <<= 1) mx = fmaxf(mx, __shfl_xor(mx, z));
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < n; j0 += M) {
        const int last = min(M, n - j0);
        const float2 ml = lane < last ? *(const float2 *)(part_ml + (at + j0 + lane) * 2)
                                      : make_float2(-INFINITY, 0.0f);
        const float c = __builtin_amdgcn_exp2f(ml.x - mx);
        total = fmaf(ml.y, c, total);
        for (int j = 0; j < last; j += 8 * G) {
            float4 x[8];
#pragma unroll
            for (int k = 0; k < 8; k++)
                x[k] = *(const float4 *)(part_acc +
                                         (at + j0 + min(j + k * G + share, last - 1)) * D + d);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float w = __shfl(c, min(j + k * G + share, M - 1), M);
                if (j + k * G + share >= last) continue;
                o.x = fmaf(x[k].x, w, o.x);
                o.y = fmaf(x[k].y, w, o.y);
                o.z = fmaf(x[k].z, w, o.z);
                o.w = fmaf(x[k].w, w, o.w);
            }
        }
    }
#pragma unroll
    for (int z = 1; z < M; z <<= 1) total += __shfl_xor(total, z);
#pragma unroll
    for (int z = L; z < M; z <<= 1) {
        o.x += __shfl_xor(o.x, z);
        o.y += __shfl_xor(o.y, z);
        o.z += __shfl_xor(o.z, z);
        o.w += __shfl_xor(o.w, z);
    }
    if (share) return;
    // A sum of 0 in a run: every block that the row sees was left out.
    if (keys || total != 0.0f) o = make_float4(o.x / total, o.y / total, o.z / total, o.w / total);
    *(float4 *)dst = o;
    flag_nonfinite(status, !(isfinite(o.x) && isfinite(o.y) && isfinite(o.z) && isfinite(o.w)));
}

}  // namespace pgpu

using namespace pgpu;

// ------------------------------------------------------------- entry points

namespace {

bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

bool cache_ok(const pgpu_kv8 *kv) {
    return kv && kv->values && kv->scales && kv->open && aligned(kv->values, 16) &&
           aligned(kv->scales, 8) && aligned(kv->open, 16) && kv->layers > 0 && kv->heads > 0 &&
           kv->heads <= 256 && (kv->head_dim == 64 || kv->head_dim == 128) && kv->blocks > 0 &&
           kv->blocks <= INT32_MAX && kv->slots > 0 && kv->slots <= INT32_MAX;
}

bool rows_ok(const pgpu_kv8_rows *r) {
    return r && r->tables && r->table_stride > 0 && r->slots && r->first && r->streams > 0 &&
           r->streams <= 65535 && r->rows >= 0 && r->max_rows >= 0 && r->max_rows <= 65535 &&
           r->max_rows <= r->rows &&
           (r->offsets ? (r->max_rows > 0 || r->rows == 0)
                       : (r->rows == r->streams && r->max_rows == 1));
}

size_t tile_bytes(const pgpu_kv8 *kv) { return (size_t)2 * kBlockPos * kv->head_dim; }

Kv8 layer_of(const pgpu_kv8 *kv, int layer) {
    const size_t tiles = (size_t)layer * kv->blocks * kv->heads;
    Kv8 x;
    x.values = kv->values + tiles * tile_bytes(kv);
    x.scales = kv->scales + tiles * 2;
    x.open = kv->open + (size_t)layer * kv->slots * kv->heads * tile_bytes(kv);
    x.heads = kv->heads;
    x.blocks = (unsigned)kv->blocks;
    x.slots = (unsigned)kv->slots;
    return x;
}

Kv8Rows rows_of(const pgpu_kv8_rows *r) {
    return {r->tables, r->table_stride, r->slots, r->first, r->offsets, r->rows, r->max_rows};
}

// Blocks that max_rows consecutive positions can lie in.
int blocks_of(int max_rows) { return (max_rows + 2 * kBlockPos - 2) / kBlockPos; }

int write_rows(const char *name, void *stream, const pgpu_kv8 *kv, int layer,
               const pgpu_kv8_rows *rows, const Kv8Turn &a, bool rotate, int *status) {
    const Kv8 c = layer_of(kv, layer);
    const int units = kv->heads * (rotate ? 2 + a.group : 2);
    const dim3 grid((units + 3) / 4, blocks_of(rows->max_rows), rows->streams);
    const Kv8Rows r = rows_of(rows);
    if (kv->head_dim == 64 && rotate)
        hipLaunchKernelGGL((k_kv8_write<64, true>), grid, dim3(256), 0, (hipStream_t)stream, c, r,
                           a, status);
    else if (kv->head_dim == 64)
        hipLaunchKernelGGL((k_kv8_write<64, false>), grid, dim3(256), 0, (hipStream_t)stream, c,
                           r, a, status);
    else if (rotate)
        hipLaunchKernelGGL((k_kv8_write<128, true>), grid, dim3(256), 0, (hipStream_t)stream, c,
                           r, a, status);
    else
        hipLaunchKernelGGL((k_kv8_write<128, false>), grid, dim3(256), 0, (hipStream_t)stream, c,
                           r, a, status);
    return launch_ok(name);
}

}  // namespace

extern "C" int pgpu_kv8_write(void *stream, const pgpu_kv8 *kv, int layer,
                              const pgpu_kv8_rows *rows, const float *k, const float *v,
                              size_t row_stride, int *status) {
    if (!cache_ok(kv) || !rows_ok(rows) || layer < 0 || layer >= kv->layers || !k || !v ||
        !status || !aligned(k, 16) || !aligned(v, 16) || row_stride % 4 != 0 ||
        row_stride < (size_t)kv->heads * kv->head_dim)
        return bad_arguments("pgpu_kv8_write");
    if (rows->rows == 0) return 1;
    Kv8Turn a = {};
    a.qkv = k;
    a.v = v;
    a.row_stride = row_stride;
    return write_rows("pgpu_kv8_write", stream, kv, layer, rows, a, false, status);
}

extern "C" int pgpu_kv8_rotate_write(void *stream, const pgpu_kv8 *kv, int layer,
                                     const pgpu_kv8_rows *rows, const float *qkv,
                                     size_t row_stride, int group, const float *q_weight,
                                     const float *k_weight, float epsilon, const float *rope,
                                     int rope_positions, float q_scale, float *q_out,
                                     int *status) {
    if (!cache_ok(kv) || !rows_ok(rows) || layer < 0 || layer >= kv->layers || !qkv || !rope ||
        !q_out || !status || !aligned(qkv, 16) || !aligned(rope, 16) || !aligned(q_out, 16) ||
        !aligned(q_weight, 16) || !aligned(k_weight, 16) || row_stride % 4 != 0 || group < 1 ||
        group > 16 || rope_positions <= 0 || !(epsilon >= 0.0f) || !__builtin_isfinite(epsilon) ||
        !__builtin_isfinite(q_scale) ||
        row_stride < (size_t)kv->heads * kv->head_dim * (2 + group))
        return bad_arguments("pgpu_kv8_rotate_write");
    if (rows->rows == 0) return 1;
    const Kv8Turn a = {qkv,     nullptr, row_stride, group,          q_weight, k_weight,
                       epsilon, rope,    rope_positions, q_scale, q_out};
    return write_rows("pgpu_kv8_rotate_write", stream, kv, layer, rows, a, true, status);
}

extern "C" int pgpu_kv8_read(void *stream, const pgpu_kv8 *kv, int layer,
                             const pgpu_kv8_rows *rows, const int32_t *lengths, float *k,
                             float *v, size_t row_stride, int *status) {
    if (!cache_ok(kv) || !rows_ok(rows) || layer < 0 || layer >= kv->layers || !lengths || !k ||
        !v || !status || !aligned(k, 16) || !aligned(v, 16) || row_stride % 4 != 0 ||
        row_stride < (size_t)kv->heads * kv->head_dim)
        return bad_arguments("pgpu_kv8_read");
    if (rows->rows == 0) return 1;
    const dim3 grid((kv->heads + 3) / 4, blocks_of(rows->max_rows), rows->streams);
    if (kv->head_dim == 64)
        hipLaunchKernelGGL(k_kv8_read<64>, grid, dim3(256), 0, (hipStream_t)stream,
                           layer_of(kv, layer), rows_of(rows), lengths, k, v, row_stride, status);
    else
        hipLaunchKernelGGL(k_kv8_read<128>, grid, dim3(256), 0, (hipStream_t)stream,
                           layer_of(kv, layer), rows_of(rows), lengths, k, v, row_stride, status);
    return launch_ok("pgpu_kv8_read");
}

extern "C" int pgpu_kv8_close(void *stream, const pgpu_kv8 *kv, int first_layer, int layers,
                              const int32_t *tables, int table_stride, const int32_t *slots,
                              const int32_t *positions, int streams, int *status) {
    if (!cache_ok(kv) || first_layer < 0 || layers <= 0 || first_layer > kv->layers - layers ||
        layers > 65535 || !tables || table_stride <= 0 || !slots || !positions || streams <= 0 ||
        streams > 65535 || !status)
        return bad_arguments("pgpu_kv8_close");
    const size_t scales = kv->blocks * kv->heads * 2, open = kv->slots * kv->heads * tile_bytes(kv),
                 values = kv->blocks * kv->heads * tile_bytes(kv);
    const dim3 grid((kv->heads + 1) / 2, layers, streams);
    if (kv->head_dim == 64)
        hipLaunchKernelGGL(k_kv8_close<64>, grid, dim3(256), 0, (hipStream_t)stream,
                           layer_of(kv, first_layer), values, scales, open, tables, table_stride,
                           slots, positions, status);
    else
        hipLaunchKernelGGL(k_kv8_close<128>, grid, dim3(256), 0, (hipStream_t)stream,
                           layer_of(kv, first_layer), values, scales, open, tables, table_stride,
                           slots, positions, status);
    return launch_ok("pgpu_kv8_close");
}

namespace {

// How an attention call deals its work: splits of `keys` keys.
struct Deal {
    int splits, keys, tiles, waves, steps;  // tiles: work-groups for a stream and head
};

Deal deal_of(const pgpu_kv8 *kv, const pgpu_kv8_rows *r, int group, int max_positions) {
    Deal d;
    if (!r->offsets) {
        // A stream's keys whole in one work-group of W waves (no parts to be joined),
        // except where few work-groups have many keys each: those are dealt to
        // work-groups of 4 waves, more keys to each the more of them there are.
        // us, whole / dealt (8 heads of 64; contexts of one stream as said, of several
        // up to that): 1 stream of 2048 keys 10.1 / 11.1, of 8187 22.4 / 10.2; 16 of
        // 2048 10.7 / 11.8, of 4096 16.2 / 14.0; 32 of 4096 18.4 / 19.4, 64 26.6 / 27.7,
        // of 6000 41.6 / 40.1; 128 of 4096 52.3 / 52.4, of 6000 81.3 / 75.6. Heads of
        // 128: 1 stream of 2048 16.0 / 11.5, 16 of 2900 22.7 / 19.1, 64 39.4 / 43.8, of
        // 8187 102 / 92.
        // Steps of a dealt work-group, 1 / 2 / 3 / 4: 4 streams of 8187 11.9 / 11.7 / 12.9
        // / 12.5, 16 19.6 / 19.4 / 20.9 / 21.4, 256 191 / 182 / 180 / 181; heads of 128
        // with 4 queries each, 24 of 8187 46.9 / 42.8 / 41.5 / 45.6, 48 of 4096 49.9 / 47.7
        // / 47.1 / 52.0, 128 126 / 124 / 115 / 127.
        // W = 4, 8, 16: 1 stream of 2048 keys 12.5, 10.4, 10.1; 32 of 4096 23.1, 18.5,
        // 18.4; 64 of 2048 17.6, 17.0, 19.5; 128 33.1, 36.6, 41.2, of 4096 56.0, 53.8,
        // 61.1; 256 of 600 24.2, 31.0, 57.6; heads of 128, 1 of 600 8.9, 8.6, 10.8, 64 of
        // 2048 31.5, 31.7, 35.1. (16 waves of 4 queries would not fit the registers.)
        d.tiles = group == 1 ? 1 : (group + 3) / 4;
        const size_t groups = (size_t)kv->heads * d.tiles * r->streams;
        const int units = (max_positions - 1) / 64 + 1;
        const bool wide = kv->head_dim != 64;
        d.waves = groups > 768 ? (units > 36 ? 8 : 4) : groups > 256 || group > 1 || wide ? 8 : 16;
        d.steps = (units + d.waves - 1) / d.waves;
        if (units > (groups < 192 ? 3 * d.waves : wide ? 48 : 80)) {
            d.waves = 4;
            d.steps = groups < 64 ? 1 : groups < 192 ? (wide ? 1 : 2) : 3;
        }
        d.keys = 64 * d.waves * d.steps;
        d.splits = (max_positions - 1) / d.keys + 1;
        return d;
    }
    // Work-groups without splits; where they are few, each row's keys are dealt
    // out until there are about two for every CU, in chunks of 64 and as many at
    // least to each as pay for the join. us, by the least chunks to a split (heads
    // of 64, 8 of them): 2 / 4 / whole: 100 rows behind 1000 keys 11.9 / 14.3 / 23.9,
    // 300 behind 200 12.9 / 14.4 / 14.2, 4 streams of 256 behind 256 17.1 / 16.2 /
    // 13.8, 1024 rows 20.5 / 18.6 / 21.7, 2 streams of 256 rows 13.1 / 10.1 / 9.9, 16
    // streams of 16 rows behind 240 12.7 / 9.3 / 9.2, behind 1000 15.5 / 15.1 / 21.2.
    d.tiles = ((r->max_rows + 15) / 16 * group + 3) / 4;
    const size_t groups = (size_t)d.tiles * kv->heads * r->streams;
    const int chunks = (max_positions - 1) / 64 + 1;
    d.splits = groups >= 512 ? 1 : (int)(1024 / groups);
    const int least = chunks <= 6 ? chunks : groups <= 64 ? 2 : chunks < 12 ? chunks : 4;
    if (d.splits > chunks / least) d.splits = chunks / least;
    if (d.splits > 32) d.splits = 32;
    d.keys = 0;
    return d;
}

template <int D>
int attend(void *stream, const Kv8 &c, const Kv8Rows &r, int streams, const Deal &d,
           const Kv8Decode &a, int *status) {
    hipStream_t st = (hipStream_t)stream;
    const int wide = c.heads * a.group;
    float *out = a.out;
    if (r.offsets) {
        const Kv8Run run = {a.q, a.q_stride, a.group, a.scale, a.max_positions, d.splits,
                            a.part_acc, a.part_ml, out, a.out_stride};
        hipLaunchKernelGGL(k_kv8_run<D>, dim3(c.heads * d.splits, d.tiles, streams), dim3(256), 0,
                           st, c, r, run, status);
    } else {
        Kv8Decode one = a;
        one.steps = d.steps;
        if (d.splits > 1) one.out = nullptr;
        const dim3 grid(c.heads * d.tiles, d.splits, streams);
#define KV8_DECODE(W, Q)                                                                        \
    hipLaunchKernelGGL((k_kv8_decode<D, W, Q>), grid, dim3(64 * W), 0, st, c, r, one, status)
        if (a.group == 1 && d.waves == 4)
            KV8_DECODE(4, 1);
        else if (a.group == 1 && d.waves == 8)
            KV8_DECODE(8, 1);
        else if (a.group == 1) {
            if constexpr (D == 64) KV8_DECODE(16, 1);
        } else if (d.waves == 4)
            KV8_DECODE(4, 4);
        else
            KV8_DECODE(8, 4);
#undef KV8_DECODE
    }
    if (!launch_ok("pgpu_kv8_attention")) return 0;
    if (d.splits == 1) return 1;
    // Many splits of few rows: a wave for each, spread over the CUs (4 streams of up
    // to 8187 keys, 32 splits: 11.8 us in all, 13.6 with 16 lanes to a head; a run of
    // 16 rows after 8000 12.0 and 14.9); else few splits of many rows.
    const size_t items = (size_t)r.max_rows * wide;
    if (d.splits >= 8 && items * streams <= 4096)
        hipLaunchKernelGGL((k_kv8_join<D, 256 / D>), dim3((unsigned)items, 1, streams), dim3(64), 0,
                           st, c, r, a.part_acc, a.part_ml, a.group, a.max_positions, d.splits,
                           d.keys, out, a.out_stride, status);
    else
        hipLaunchKernelGGL((k_kv8_join<D, 1>),
                           dim3((unsigned)((items * (D / 4) + 255) / 256), 1, streams), dim3(256),
                           0, st, c, r, a.part_acc, a.part_ml, a.group, a.max_positions, d.splits,
                           d.keys, out, a.out_stride, status);
    return launch_ok("pgpu_kv8_attention");
}

}  // namespace

extern "C" size_t pgpu_kv8_attention_bytes(const pgpu_kv8 *kv, const pgpu_kv8_rows *rows,
                                           int group, int max_positions) {
    if (!cache_ok(kv) || !rows_ok(rows) || group < 1 || group > 16 || max_positions <= 0) return 0;
    if (rows->rows == 0) return 0;
    // Fewer streams, rows or positions may be dealt to more work-groups: the most
    // parts of any of them.
    size_t parts = 0;
    if (!rows->offsets) {
        // More positions never give fewer parts. More streams do, at the numbers of
        // work-groups where the keys to each change: the streams before those count.
        const int heads = kv->heads * (group == 1 ? 1 : (group + 3) / 4);
        for (int n : {rows->streams, 63 / heads, 191 / heads}) {
            pgpu_kv8_rows fewer = *rows;
            fewer.streams = n;
            if (n < 1 || n > rows->streams) continue;
            const Deal d = deal_of(kv, &fewer, group, max_positions);
            if (d.splits > 1) parts = std::max(parts, (size_t)n * kv->heads * group * d.splits);
        }
    } else {
        // Splits times work-groups are at most 1024, a work-group has 64 rows.
        const int chunks = (max_positions - 1) / 64 + 1;
        const int most = std::min({32, chunks <= 6 ? 1 : chunks / 2,
                                   1024 / (kv->heads * ((group + 3) / 4))});
        if (most > 1)
            parts = std::min((size_t)1024 * 64, (size_t)rows->streams * rows->max_rows *
                                                    kv->heads * group * most);
    }
    return parts * (kv->head_dim + 2) * sizeof(float);
}

extern "C" int pgpu_kv8_attention(void *stream, const pgpu_kv8 *kv, int layer,
                                  const pgpu_kv8_rows *rows, const float *q, size_t q_stride,
                                  int group, float scale, int max_positions, float *out,
                                  size_t out_stride, void *work, size_t work_bytes,
                                  int *status) {
    constexpr float kLog2e = 1.44269504f;
    const size_t width = kv ? (size_t)kv->heads * kv->head_dim * group : 0;
    if (!cache_ok(kv) || !rows_ok(rows) || layer < 0 || layer >= kv->layers || !q || !out ||
        !status || !aligned(q, 16) || !aligned(out, 16) || q_stride % 4 != 0 ||
        out_stride % 4 != 0 || group < 1 || group > 16 || q_stride < width ||
        out_stride < width || max_positions <= 0 || !__builtin_isfinite(scale * kLog2e))
        return bad_arguments("pgpu_kv8_attention");
    if (rows->rows == 0) return 1;
    const Deal d = deal_of(kv, rows, group, max_positions);
    // The grid's limit: 16 million positions of one row a stream.
    if (d.splits > 65535) return bad_arguments("pgpu_kv8_attention");
    const size_t parts = d.splits > 1 ? (size_t)rows->streams * rows->max_rows * kv->heads *
                                            group * d.splits : 0;
    if (parts && (!work || !aligned(work, 16) ||
                  work_bytes < parts * (kv->head_dim + 2) * sizeof(float)))
        return bad_arguments("pgpu_kv8_attention (workspace)");
    const Kv8Decode a = {q, q_stride, group, scale * kLog2e, max_positions, d.splits, 1,
                         (float *)work, (float *)work + parts * kv->head_dim, out, out_stride};
    const Kv8 c = layer_of(kv, layer);
    return kv->head_dim == 64
               ? attend<64>(stream, c, rows_of(rows), rows->streams, d, a, status)
               : attend<128>(stream, c, rows_of(rows), rows->streams, d, a, status);
}
