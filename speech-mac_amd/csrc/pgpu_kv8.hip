// 8-bit paged KV cache: quantised writes (with the heads' norm and rotation in
// the same pass), reads, and causal attention over it. The formats and the
// rules of the stored values are in phonon_gpu.h.
#include "pgpu_common.hpp"
#include "phonon_gpu.h"

namespace pgpu {

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
    x.first = r.first[s];
    x.slot = r.slots[s];
    x.row0 = r.offsets ? r.offsets[s] : s;
    const int end = r.offsets ? r.offsets[s + 1] : s + 1;
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

// ------------------------------------------------------------------- writing

// A work-group of 256 threads holds one (block, head): thread u the NV groups
// of 4 dims at elements 4 (256 i + u) of [16][D], of keys and of values.
template <int D>
struct Kv8Tile {
    static constexpr int NV = D / 64;
    float4 x[2][NV];
};

template <int D>
struct Kv8Shared {
    float top[2][4];
    __align__(16) int8_t values[kBlockPos * D];
};

// The block's 16 rows in x -> the cache. Every thread of the work-group calls
// it. A non-finite value: a NaN scale, and status bit 1.
template <int D>
__device__ inline void kv8_store(const Kv8 &kv, unsigned block, int head, const Kv8Tile<D> &t,
                                 Kv8Shared<D> &sh, int *status) {
    constexpr int NV = D / 64;
    const int u = threadIdx.x, wave = u >> 6;
    float top[2];
#pragma unroll
    for (int p = 0; p < 2; p++) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const float4 v = t.x[p][i];
            // |x| orders like its bits: infinities and NaN come out on top.
            m = bitsf(max(max(fbits(m), fbits(v.x) & 0x7fffffffu),
                          max(fbits(v.y) & 0x7fffffffu,
                              max(fbits(v.z) & 0x7fffffffu, fbits(v.w) & 0x7fffffffu))));
        }
        uint32_t b = fbits(m);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) b = max(b, (uint32_t)__shfl_xor((int)b, o));
        top[p] = bitsf(b);
    }
    if ((u & 63) == 0) {
        sh.top[0][wave] = top[0];
        sh.top[1][wave] = top[1];
    }
    __syncthreads();
    int8_t *tile = kv.values + kv8_tile<D>(kv, block, head);
    float scale[2];
    bool bad = false;
#pragma unroll
    for (int p = 0; p < 2; p++) {
        uint32_t b = 0;
        for (int w = 0; w < 4; w++) b = max(b, fbits(sh.top[p][w]));
        const bool wild = b >= 0x7f800000u;
        bad |= wild;
        const float s = kv8_scale(bitsf(b));
        scale[p] = wild ? __builtin_nanf("") : s;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int e = (i * 256 + u) * 4, j = e / D, d = e % D;
            const float4 v = t.x[p][i];
            const float f[4] = {v.x, v.y, v.z, v.w};
            int8_t q[4];
#pragma unroll
            for (int k = 0; k < 4; k++)
                q[k] = wild ? (int8_t)0 : (int8_t)(int)rintf(f[k] / s);
            if (p == 0) {
                *(char4 *)(tile + e) = make_char4(q[0], q[1], q[2], q[3]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) sh.values[kv8_value_at<D>(j, d + k)] = q[k];
            }
        }
    }
    __syncthreads();
    if (u < D) *(int4 *)(tile + kBlockPos * D + u * 16) = *(const int4 *)(sh.values + u * 16);
    if (u == 0)
        *(float2 *)(kv.scales + ((size_t)block * kv.heads + head) * 2) =
            make_float2(scale[0], scale[1]);
    if (bad && u == 0) atomicOr(status, 1);
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

// 4 dims of a row's head: normalised (weight), turned, scaled; in 64 bits,
// rounded once. The D / 4 lanes of a row are neighbours in a wave, and all
// lanes of the wave call it.
template <int D>
__device__ inline float4 kv8_turn(float4 x, int d, const float *weight, float epsilon,
                                  const float *rope_row, float scale) {
    double y[4] = {x.x, x.y, x.z, x.w};
    if (weight) {
        double sq = y[0] * y[0] + y[1] * y[1] + y[2] * y[2] + y[3] * y[3];
#pragma unroll
        for (int o = 1; o < D / 4; o <<= 1) sq += __shfl_xor(sq, o);
        const double r = 1.0 / sqrt(sq / D + (double)epsilon);
        const float4 w = *(const float4 *)(weight + d);
        y[0] = y[0] * r * w.x;
        y[1] = y[1] * r * w.y;
        y[2] = y[2] * r * w.z;
        y[3] = y[3] * r * w.w;
    }
    const float4 cs = *(const float4 *)(rope_row + d);
    const double f = scale;
    return make_float4((float)((y[0] * cs.x - y[1] * cs.y) * f),
                       (float)((y[0] * cs.y + y[1] * cs.x) * f),
                       (float)((y[2] * cs.z - y[3] * cs.w) * f),
                       (float)((y[2] * cs.w + y[3] * cs.z) * f));
}

// One (block of the call's rows, head) per work-group: y < heads keys and
// values, past them (rotate) query head y - heads.
template <int D, bool ROTATE>
__global__ __launch_bounds__(256) void k_kv8_write(Kv8 kv, Kv8Rows rows, Kv8Turn a, int *status) {
    constexpr int NV = D / 64;
    __shared__ Kv8Shared<D> sh;
    const int s = blockIdx.z, u = threadIdx.x;
    const bool queries = ROTATE && (int)blockIdx.y >= kv.heads;
    const Kv8Span span = kv8_span(kv, rows, s, ROTATE ? a.rope_positions : INT32_MAX - kBlockPos,
                                  u == 0 && blockIdx.x == 0 && blockIdx.y == 0, status);
    if (!span.live) return;
    const int end = span.first + span.count;
    const int block = span.first / kBlockPos + (int)blockIdx.x, newest = (end - 1) / kBlockPos;
    if (block > newest) return;
    const int head = queries ? (int)blockIdx.y - kv.heads : (int)blockIdx.y;
    bool bad = false;

    if constexpr (ROTATE) {
        if (queries) {
            const int width = kv.heads * a.group * D;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int e = (i * 256 + u) * 4, d = e % D, p = block * kBlockPos + e / D;
                const bool in = p >= span.first && p < end;
                const size_t row = (size_t)(span.row0 + (in ? p - span.first : 0));
                float4 x = *(const float4 *)(a.qkv + row * a.row_stride + head * D + d);
                x = kv8_turn<D>(x, d, a.q_weight, a.epsilon,
                                a.rope + (size_t)(in ? p : span.first) * D, a.q_scale);
                if (in) {
                    *(float4 *)(a.q_out + row * width + head * D + d) = x;
                    bad |= !(isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w));
                }
            }
            flag_nonfinite(status, bad);
            return;
        }
    }

    float *slot = kv.open + ((size_t)span.slot * kv.heads + head) * (2 * kBlockPos * D);
    // Rows of block b (the keys and values of this thread's places): the
    // call's, else what the slot held (only before the call's first row), else 0.
    auto gather = [&](int b, Kv8Tile<D> &t) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int e = (i * 256 + u) * 4, d = e % D, p = b * kBlockPos + e / D;
            const bool in = p >= span.first && p < end;
            const size_t row = (size_t)(span.row0 + (in ? p - span.first : 0));
            if constexpr (ROTATE) {
                const float *src = a.qkv + row * a.row_stride;
                float4 k = *(const float4 *)(src + (kv.heads * a.group + head) * D + d);
                t.x[0][i] = kv8_turn<D>(k, d, a.k_weight, a.epsilon,
                                        a.rope + (size_t)(in ? p : span.first) * D, 1.0f);
                t.x[1][i] = *(const float4 *)(src + (kv.heads * (a.group + 1) + head) * D + d);
            } else {
                t.x[0][i] = *(const float4 *)(a.qkv + row * a.row_stride + head * D + d);
                t.x[1][i] = *(const float4 *)(a.v + row * a.row_stride + head * D + d);
            }
            if (!in)
#pragma unroll
                for (int k = 0; k < 2; k++)
                    t.x[k][i] = p < span.first ? *(const float4 *)(slot + k * kBlockPos * D + e)
                                               : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    // The call's rows of block b into the slot.
    auto keep = [&](int b, const Kv8Tile<D> &t) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int e = (i * 256 + u) * 4, p = b * kBlockPos + e / D;
            if (p < span.first || p >= end) continue;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float4 x = t.x[k][i];
                *(float4 *)(slot + k * kBlockPos * D + e) = x;
                bad |= !(isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w));
            }
        }
    };
    Kv8Tile<D> t;
    gather(block, t);
    if ((block + 1) * kBlockPos <= end) {
        const int id = rows.tables[(size_t)s * rows.table_stride + block];
        if ((unsigned)id < kv.blocks)
            kv8_store<D>(kv, (unsigned)id, head, t, sh, status);
        else if (u == 0)
            atomicOr(status, 2);
    }
    // The first block's work-group, which reads the slot's earlier rows, also
    // replaces them: its threads have all read them by then.
    if (blockIdx.x != 0) return;
    __syncthreads();
    if (block != newest) gather(newest, t);
    keep(newest, t);
    flag_nonfinite(status, bad);
}

// The open slots' full blocks -> the cache. Layers and streams in z.
template <int D>
__global__ __launch_bounds__(256) void k_kv8_close(Kv8 kv, size_t layer_values,
                                                   size_t layer_scales, size_t layer_open,
                                                   const int32_t *tables, int table_stride,
                                                   const int32_t *slots, const int32_t *positions,
                                                   int *status) {
    __shared__ Kv8Shared<D> sh;
    const int s = blockIdx.z, head = blockIdx.x, layer = blockIdx.y, u = threadIdx.x;
    const int p = positions[s];
    if (p < 0 || p % kBlockPos != kBlockPos - 1) return;
    const int id = p / kBlockPos < table_stride
                       ? tables[(size_t)s * table_stride + p / kBlockPos] : -1;
    const int slot = slots[s];
    if ((unsigned)id >= kv.blocks || (unsigned)slot >= kv.slots) {
        if (u == 0) atomicOr(status, 2);
        return;
    }
    kv.values += layer * layer_values;
    kv.scales += layer * layer_scales;
    const float *src = kv.open + layer * layer_open +
                       ((size_t)slot * kv.heads + head) * (2 * kBlockPos * D);
    Kv8Tile<D> t;
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < D / 64; i++)
            t.x[k][i] = *(const float4 *)(src + k * kBlockPos * D + (i * 256 + u) * 4);
    kv8_store<D>(kv, (unsigned)id, head, t, sh, status);
}

// ------------------------------------------------------------------- reading

template <int D>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8 kv, Kv8Rows rows, const int32_t *lengths,
                                                  float *k, float *v, size_t row_stride,
                                                  int *status) {
    constexpr int NV = D / 64;
    __shared__ __align__(16) int8_t sh[kBlockPos * D];
    const int s = blockIdx.z, head = blockIdx.y, u = threadIdx.x;
    const Kv8Span span = kv8_span(kv, rows, s, lengths[s],
                                  u == 0 && blockIdx.x == 0 && head == 0, status);
    if (!span.live) return;
    const int end = span.first + span.count;
    const int block = span.first / kBlockPos + (int)blockIdx.x;
    if (block * kBlockPos >= end) return;
    const bool open = block == (lengths[s] - 1) / kBlockPos;
    const float *slot = kv.open + ((size_t)span.slot * kv.heads + head) * (2 * kBlockPos * D);
    const int8_t *tile = nullptr;
    float2 scale = make_float2(1.0f, 1.0f);
    if (!open) {
        const int id = rows.tables[(size_t)s * rows.table_stride + block];
        if ((unsigned)id >= kv.blocks) {
            if (u == 0) atomicOr(status, 2);
            return;
        }
        tile = kv.values + kv8_tile<D>(kv, (unsigned)id, head);
        scale = *(const float2 *)(kv.scales + ((size_t)id * kv.heads + head) * 2);
        if (u < D) *(int4 *)(sh + u * 16) = *(const int4 *)(tile + kBlockPos * D + u * 16);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int e = (i * 256 + u) * 4, j = e / D, d = e % D, p = block * kBlockPos + j;
        if (p < span.first || p >= end) continue;
        float4 x, y;
        if (open) {
            x = *(const float4 *)(slot + e);
            y = *(const float4 *)(slot + kBlockPos * D + e);
        } else {
            const char4 q = *(const char4 *)(tile + e);
            x = make_float4(q.x * scale.x, q.y * scale.x, q.z * scale.x, q.w * scale.x);
            y = make_float4(sh[kv8_value_at<D>(j, d)] * scale.y,
                            sh[kv8_value_at<D>(j, d + 1)] * scale.y,
                            sh[kv8_value_at<D>(j, d + 2)] * scale.y,
                            sh[kv8_value_at<D>(j, d + 3)] * scale.y);
        }
        const size_t at = (size_t)(span.row0 + p - span.first) * row_stride + head * D + d;
        *(float4 *)(k + at) = x;
        *(float4 *)(v + at) = y;
    }
}

// ----------------------------------------------------------------- attention

// One wave per (row, query head), a block of 16 keys at a time: lane l takes
// key l % 16 and the quarter l / 16 of the dims for the score, then dims l
// (and l + 64) of the values.
template <int D>
__global__ __launch_bounds__(64) void k_kv8_attend(Kv8 kv, Kv8Rows rows, const float *q,
                                                   size_t q_stride, int group, float scale,
                                                   int max_positions, float *out,
                                                   size_t out_stride, int *status) {
    constexpr int N = D / 64;
    const int s = blockIdx.z, qh = blockIdx.y, i = blockIdx.x, lane = threadIdx.x;
    const Kv8Span span = kv8_span(kv, rows, s, max_positions,
                                  lane == 0 && i == 0 && qh == 0, status);
    if (i >= span.count) return;
    const size_t row = (size_t)(span.row0 + i);
    float *dst = out + row * out_stride + qh * D + lane;
    if (!span.live) {
        if (span.first < 0)
            for (int n = 0; n < N; n++) dst[n * 64] = 0.0f;
        return;
    }
    const int head = qh / group, key = lane & 15, part = lane >> 4;
    const int p = span.first + i, newest = (span.first + span.count - 1) / kBlockPos;
    const float *qr = q + row * q_stride + qh * D + part * (D / 4);
    float w[D / 4];
#pragma unroll
    for (int d = 0; d < D / 4; d++) w[d] = qr[d] * scale;
    float m = -INFINITY, l = 0.0f, acc[N] = {};
    for (int b = 0; b <= p / kBlockPos; b++) {
        float dot = 0.0f, val[N][kBlockPos];
        if (b == newest) {
            const float *slot = kv.open + ((size_t)span.slot * kv.heads + head) *
                                              (2 * kBlockPos * D);
            for (int d = 0; d < D / 4; d++)
                dot = fmaf(w[d], slot[key * D + part * (D / 4) + d], dot);
            for (int n = 0; n < N; n++)
                for (int j = 0; j < kBlockPos; j++)
                    val[n][j] = slot[kBlockPos * D + j * D + n * 64 + lane];
        } else {
            const int id = rows.tables[(size_t)s * rows.table_stride + b];
            if ((unsigned)id >= kv.blocks) {
                if (lane == 0) atomicOr(status, 2);
                return;
            }
            const int8_t *tile = kv.values + kv8_tile<D>(kv, (unsigned)id, head);
            const float2 sc =
                *(const float2 *)(kv.scales + ((size_t)id * kv.heads + head) * 2);
            for (int d = 0; d < D / 4; d++)
                dot = fmaf(w[d], (float)tile[key * D + part * (D / 4) + d], dot);
            dot *= sc.x;
            for (int n = 0; n < N; n++)
                for (int j = 0; j < kBlockPos; j++)
                    val[n][j] =
                        sc.y * (float)tile[kBlockPos * D + kv8_value_at<D>(j, n * 64 + lane)];
        }
        dot = xor16_32_sum(dot);
        const int keys = min(kBlockPos, p + 1 - b * kBlockPos);
        float top = key < keys ? dot : -INFINITY;
        for (int o = 8; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float mx = fmaxf(m, top), keep = expf(m - mx);
        m = mx;
        l *= keep;
        for (int n = 0; n < N; n++) acc[n] *= keep;
        for (int j = 0; j < kBlockPos; j++) {
            // Rows past the position may hold anything: skipped, not weighted.
            if (j >= keys) break;
            const float e = expf(__shfl(dot, j) - m);
            l += e;
            for (int n = 0; n < N; n++) acc[n] = fmaf(e, val[n][j], acc[n]);
        }
    }
    bool bad = false;
    for (int n = 0; n < N; n++) {
        const float o = acc[n] / l;
        dst[n * 64] = o;
        bad |= !isfinite(o);
    }
    flag_nonfinite(status, bad);
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
           r->streams <= 65535 && r->rows >= 0 && r->max_rows >= 0 && r->max_rows <= r->rows &&
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
    const dim3 grid(blocks_of(rows->max_rows), kv->heads * (rotate ? 1 + a.group : 1),
                    rows->streams);
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
    const dim3 grid(blocks_of(rows->max_rows), kv->heads, rows->streams);
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
    const dim3 grid(kv->heads, layers, streams);
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

extern "C" size_t pgpu_kv8_attention_bytes(const pgpu_kv8 *, const pgpu_kv8_rows *, int, int) {
    return 0;
}

extern "C" int pgpu_kv8_attention(void *stream, const pgpu_kv8 *kv, int layer,
                                  const pgpu_kv8_rows *rows, const float *q, size_t q_stride,
                                  int group, float scale, int max_positions, float *out,
                                  size_t out_stride, void *work, size_t work_bytes,
                                  int *status) {
    const size_t width = kv ? (size_t)kv->heads * kv->head_dim * group : 0;
    if (!cache_ok(kv) || !rows_ok(rows) || layer < 0 || layer >= kv->layers || !q || !out ||
        !status || !aligned(q, 16) || !aligned(out, 16) || q_stride % 4 != 0 ||
        out_stride % 4 != 0 || group < 1 || group > 16 || q_stride < width ||
        out_stride < width || max_positions <= 0 || !__builtin_isfinite(scale))
        return bad_arguments("pgpu_kv8_attention");
    if (rows->rows == 0) return 1;
    const dim3 grid(rows->max_rows, kv->heads * group, rows->streams);
    if (kv->head_dim == 64)
        hipLaunchKernelGGL(k_kv8_attend<64>, grid, dim3(64), 0, (hipStream_t)stream,
                           layer_of(kv, layer), rows_of(rows), q, q_stride, group, scale,
                           max_positions, out, out_stride, status);
    else
        hipLaunchKernelGGL(k_kv8_attend<128>, grid, dim3(64), 0, (hipStream_t)stream,
                           layer_of(kv, layer), rows_of(rows), q, q_stride, group, scale,
                           max_positions, out, out_stride, status);
    return launch_ok("pgpu_kv8_attention");
}
