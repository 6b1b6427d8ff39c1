// 4-bit paged KV cache: quantised writes, reads, causal attention over it with
// the sums of its weights, and eviction by them. The formats and the rules of the
// stored values are in phonon_gpu.h.
#include <algorithm>

#include "pgpu_kv.hpp"
#include "phonon_gpu.h"

namespace pgpu {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kSpan = 64;         // dims of a scale
constexpr int kPlane = 512;       // bytes of a block's 64 dims, of keys or of values
constexpr float kLeastScale = 0x1p-17f, kMostScale = 8160.0f;
constexpr int kMostRows = 1 << 30;  // of a stream: a block past its last is an int32 still
// With one row a stream: the grid's 65535 splits of the fewest keys that one has.
constexpr int kMostOne = 65535 * 256;

// One layer of the cache, and the rows of a call (pgpu_kv4, pgpu_kv4_rows).
struct Kv4 {
    uint8_t *values;
    uint32_t *scales;  // (key, value) pairs
    int heads;
    unsigned blocks;
};

struct Kv4Rows {
    const int32_t *tables;
    int table_stride;
    const int32_t *first, *offsets;
    int rows, max_rows;
};

// A stream's rows, checked: uniform over the work-group.
struct Kv4Span {
    int first, count, row0;
    bool live;
};

// limit: indexes must be below it, and below kMostRows. A stream that breaks a bound is flagged (by
// the thread with `speak`) and left out.
__device__ inline Kv4Span kv4_span(const Kv4Rows &r, int s, int limit, bool speak, int *status) {
    Kv4Span x;
    x.first = uniform_load(r.first + s);
    x.row0 = r.offsets ? uniform_load(r.offsets + s) : s;
    const int end = r.offsets ? uniform_load(r.offsets + s + 1) : s + 1;
    // 64 bits: any int32 may stand in the arrays.
    const long long count = (long long)end - x.row0;
    const bool wild = x.row0 < 0 || count < 0 || end > r.rows || count > r.max_rows;
    x.count = wild ? 0 : (int)count;
    const long long last = (long long)x.first + x.count;
    const bool bad = wild || (x.first >= 0 && x.count > 0 &&
                              (last > min(limit, kMostRows) || last > (long long)r.table_stride * kBlockPos));
    x.live = !bad && x.first >= 0 && x.count > 0;
    if (bad && speak) atomicOr(status, 2);
    return x;
}

// Bytes of a (block, head); its values start half way. And its scales.
template <int D>
__device__ inline uint8_t *kv4_tile(const Kv4 &kv, unsigned block, int head) {
    return kv.values + ((size_t)block * kv.heads + head) * (D * kBlockPos);
}
template <int D>
__device__ inline uint32_t *kv4_scales(const Kv4 &kv, unsigned block, int head) {
    return kv.scales + ((size_t)block * kv.heads + head) * (D / kSpan * kBlockPos);
}
__device__ inline float key_scale(uint32_t pair) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)pair);
}
__device__ inline float value_scale(uint32_t pair) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(pair >> 16));
}
// Number i of the eight in a word: 4 h + b is half h of byte b.
__device__ inline float nibble(uint32_t w, int i) {
    const int at = (i & 3) * 8 + (i >> 2) * 4;
    return (float)((int)(w << (28 - at)) >> 28);
}

// ------------------------------------------------------------------- writing

// max x, max -x of 64 dims -> their scale. Eight significant bits: see phonon_gpu.h.
__device__ inline float kv4_scale(float top, float bottom) {
    const uint32_t bits = fbits(fmaxf(fmaxf(top / 7.0f, bottom / 8.0f), 0.0f)) + 0xFFFFu;
    return fmaxf(bitsf(bits & ~0xFFFFu), kLeastScale);
}

__device__ inline uint32_t xor1(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false);
}
// The largest of a quad's lanes; NaN if one is NaN.
__device__ inline float quad_largest(float x) {
    x = __builtin_elementwise_maximum(x, bitsf(xor1(fbits(x))));
    return __builtin_elementwise_maximum(
        x, bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(x), 0x4E, 0xf, 0xf, false)));
}
// Of 8 lanes, the first four get the last ones' and the other way round.
__device__ inline float other_quad(float x) {
    return bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(x), 0x141, 0xf, 0xf, false));
}

// Eight dims of a row -> whole numbers, the low bytes of q. x / s by the reciprocal, which
// is off by less than 2^-20 below 8; where that could decide a rounding, by the division.
__device__ inline void kv4_round(const float4 (&x)[2], float s, float inverse, uint32_t (&q)[2][4]) {
    constexpr float kWhole = 0x1.8p23f;  // a sum with it is a whole number in the last bits
    float off = 0.0f;
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int z = 0; z < 4; z++) {
            const float f = (&x[e].x)[z], sum = fmaf(f, inverse, kWhole);
            off = fmaxf(off, fabsf(fmaf(f, inverse, -(sum - kWhole))));
            q[e][z] = fbits(sum);
        }
    if (off > 0.5f - 2e-6f)
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int z = 0; z < 4; z++) q[e][z] = fbits((&x[e].x)[z] / s + kWhole);
}

// Four low bytes side by side.
__device__ inline uint32_t low_bytes(const uint32_t (&q)[4]) {
    return __builtin_amdgcn_perm(q[1], q[0], 0x0C0C0400u) | __builtin_amdgcn_perm(q[3], q[2], 0x04000C0Cu);
}

// The bits of 16 numbers' 8 bytes that rows lo .. hi - 1 take.
__device__ inline uint64_t row_bits(int lo, int hi) {
    uint64_t m = 0;
#pragma unroll
    for (int j = 0; j < kBlockPos; j++)
        if (j >= lo && j < hi) m |= (uint64_t)15 << ((j >> 3) * 32 + (j & 3) * 8 + (j >> 2 & 1) * 4);
    return m;
}

// A wave for each (block of the call's rows, head). Lane (g, c) has rows 2 g and 2 g + 1,
// of every 64 dims 4 c .. 4 c + 3 and 32 + those: eight lanes share a row, and each half
// of them finds one of the two rows' scales. Keys are packed as they lie. Values change
// from rows to dims through LDS, four numbers a word. Bound by the rows' bytes: 64 streams
// of up to 2048 rows, 8 heads of 64, 277 MB in 54 us. A row's 128 bytes to an instruction
// are whole cache lines (64, with 4 lanes a row: 76 us); 256 with 16 lanes a row, each with
// its scales, are bound by the vector units (65). 211 rows of 1 stream 3.8 us, 5.9 so.
template <int D>
__global__ __launch_bounds__(256) void k_kv4_write(Kv4 kv, Kv4Rows rows, const float *k,
                                                   const float *v, size_t row_stride,
                                                   int *status) {
    constexpr int N = D / kSpan;
    __shared__ __align__(16) uint32_t lds[4][N][16][kBlockPos];  // [wave][64 dims][4 dims][row]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int s = blockIdx.z, head = blockIdx.x * 4 + wave, g = lane >> 3, c = lane & 7;
    const Kv4Span span = kv4_span(rows, s, kMostRows,
                                  threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0, status);
    if (!span.live || head >= kv.heads) return;
    const int end = span.first + span.count, block = span.first / kBlockPos + (int)blockIdx.y;
    if (block * kBlockPos >= end) return;
    const int id = uniform_load(rows.tables + (size_t)s * rows.table_stride + block);
    const int lo = max(span.first - block * kBlockPos, 0), hi = min(end - block * kBlockPos, 16);
    float4 x[2][N][2][2];  // keys, values; 64 dims; row; 32 dims
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const int j = g * 2 + r;
        const bool in = j >= lo && j < hi;
        const size_t at = (size_t)(span.row0 + (in ? block * kBlockPos + j - span.first : 0)) *
                              row_stride + (size_t)head * D + c * 4;
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
                x[0][n][r][e] = in ? once_load(k + at + n * kSpan + e * 32) : none;
                x[1][n][r][e] = in ? once_load(v + at + n * kSpan + e * 32) : none;
            }
    }
    if ((unsigned)id >= kv.blocks) {
        if (lane == 0) atomicOr(status, 2);
        return;
    }
    const int half = c >> 2;  // this lane finds row 2 g + half's scales
    float mine[2][N];
    bool wild = false;
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
        for (int n = 0; n < N; n++) {
            float top[2], bottom[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                top[r] = -INFINITY, bottom[r] = INFINITY;
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int z = 0; z < 4; z++) {
                        const float f = (&x[p][n][r][e].x)[z];
                        top[r] = __builtin_elementwise_maximum(top[r], f);
                        bottom[r] = __builtin_elementwise_minimum(bottom[r], f);
                    }
            }
            const float t = quad_largest(__builtin_elementwise_maximum(
                half ? top[1] : top[0], other_quad(half ? top[0] : top[1])));
            const float b = -quad_largest(-__builtin_elementwise_minimum(
                half ? bottom[1] : bottom[0], other_quad(half ? bottom[0] : bottom[1])));
            mine[p][n] = kv4_scale(t, -b);
            wild |= !(t < INFINITY && b > -INFINITY && mine[p][n] <= kMostScale);
        }
    uint8_t *tile = kv4_tile<D>(kv, (unsigned)id, head);
    uint32_t *scales = kv4_scales<D>(kv, (unsigned)id, head);
    const float keep = wild ? 0.0f : 1.0f, keep2 = other_quad(keep);
    const uint32_t nibbles[2] = {(half ? keep2 : keep) != 0.0f ? 0x0F0F0F0Fu : 0u,
                                 (half ? keep : keep2) != 0.0f ? 0x0F0F0F0Fu : 0u};
    const int odd = c & 1;
#pragma unroll
    for (int n = 0; n < N; n++) {
        uint32_t w[2][2][2];  // keys, values; row; 32 dims
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const float inverse = 1.0f / mine[p][n];
            const float s2 = other_quad(mine[p][n]), inverse2 = other_quad(inverse);
#pragma unroll
            for (int r = 0; r < 2; r++) {
                uint32_t q[2][4];
                kv4_round(x[p][n][r], half == r ? mine[p][n] : s2, half == r ? inverse : inverse2, q);
#pragma unroll
                for (int e = 0; e < 2; e++) w[p][r][e] = low_bytes(q[e]) & nibbles[r];
            }
        }
        // Keys: four dims are half of a word, the next lane's the other half.
        const int j = g * 2 + odd;
        const bool in = j >= lo && j < hi;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t w0 = w[0][0][e] << (odd * 4), w1 = w[0][1][e] << (odd * 4);
            const uint32_t word = (odd ? w1 : w0) | xor1(odd ? w0 : w1);
            if (in) *(uint32_t *)(tile + n * kPlane + j * (kSpan / 2) + e * 16 + (c >> 1) * 4) = word;
            *(uint2 *)&lds[wave][n][e * 8 + c][g * 2] = make_uint2(w[1][0][e], w[1][1][e]);
        }
        if ((c & 3) == 0 && g * 2 + half >= lo && g * 2 + half < hi) {
            const auto pair = __builtin_amdgcn_cvt_pkrtz(mine[0][n], mine[1][n]);
            scales[n * kBlockPos + g * 2 + half] =
                wild ? 0x7E007E00u : __builtin_bit_cast(uint32_t, pair);
        }
    }
    wave_lds_fence();
    // Values: lane (d, a) has rows 4 a .. 4 a + 3 of dims 4 d .. 4 d + 3, half of a word, the
    // next lane's the other half.
    const int d = lane >> 2, a = lane & 3;
    const uint64_t there = row_bits(lo, hi);
    const uint32_t bits = (uint32_t)(a < 2 ? there : there >> 32);
#pragma unroll
    for (int n = 0; n < N; n++) {
        const uint4 r = *(const uint4 *)&lds[wave][n][d][a * 4];
        const uint32_t a0 = __builtin_amdgcn_perm(r.y, r.x, 0x05010400u);
        const uint32_t a1 = __builtin_amdgcn_perm(r.y, r.x, 0x07030602u);
        const uint32_t b0 = __builtin_amdgcn_perm(r.w, r.z, 0x05010400u);
        const uint32_t b1 = __builtin_amdgcn_perm(r.w, r.z, 0x07030602u);
        const uint32_t dim[4] = {__builtin_amdgcn_perm(b0, a0, 0x05040100u),
                                 __builtin_amdgcn_perm(b0, a0, 0x07060302u),
                                 __builtin_amdgcn_perm(b1, a1, 0x05040100u),
                                 __builtin_amdgcn_perm(b1, a1, 0x07060302u)};
        uint32_t *to = (uint32_t *)(tile + (N + n) * kPlane + (d * 4 + odd * 2) * 8) + (a >> 1);
#pragma unroll
        for (int z = 0; z < 2; z++) {
            const uint32_t w0 = dim[z] << (odd * 4), w1 = dim[z + 2] << (odd * 4);
            uint32_t word = (odd ? w1 : w0) | xor1(odd ? w0 : w1);
            if (~bits) word = (to[z * 2] & ~bits) | (word & bits);
            to[z * 2] = word;
        }
    }
    flag_nonfinite(status, wild);
}

// ------------------------------------------------------------------- reading

// A wave for each (block of the rows read, head). Bound by the fp32 rows that it writes: 64
// streams of up to 1024 rows, 8 heads of 64, 258 MB in 43 us.
template <int D>
__global__ __launch_bounds__(256) void k_kv4_read(Kv4 kv, Kv4Rows rows, const int32_t *lengths,
                                                  float *k, float *v, size_t row_stride,
                                                  int *status) {
    constexpr int N = D / kSpan;
    __shared__ __align__(16) uint32_t lds[4][kSpan * 2];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int s = blockIdx.z, head = blockIdx.x * 4 + wave, g = lane >> 4, c = lane & 15;
    const Kv4Span span = kv4_span(rows, s, uniform_load(lengths + s),
                                  threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0, status);
    if (!span.live || head >= kv.heads) return;
    const int end = span.first + span.count, block = span.first / kBlockPos + (int)blockIdx.y;
    if (block * kBlockPos >= end) return;
    const int id = uniform_load(rows.tables + (size_t)s * rows.table_stride + block);
    if ((unsigned)id >= kv.blocks) {
        if (lane == 0) atomicOr(status, 2);
        return;
    }
    const uint8_t *tile = kv4_tile<D>(kv, (unsigned)id, head);
    const uint32_t *scales = kv4_scales<D>(kv, (unsigned)id, head);
    uint32_t keys[N][4], pairs[N][4];
    uint64_t dim[N];
#pragma unroll
    for (int n = 0; n < N; n++) {
        dim[n] = *((const uint64_t *)(tile + (N + n) * kPlane) + lane);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            keys[n][r] = *(const uint32_t *)(tile + n * kPlane + (g * 4 + r) * (kSpan / 2) + (c >> 1) * 4);
            pairs[n][r] = scales[n * kBlockPos + g * 4 + r];
        }
    }
#pragma unroll
    for (int n = 0; n < N; n++) {
        *(uint64_t *)&lds[wave][lane * 2] = dim[n];
        wave_lds_fence();
        uint32_t w[4];  // of dim z: the eight rows of which four are this lane's
#pragma unroll
        for (int z = 0; z < 4; z++) w[z] = lds[wave][(c * 4 + z) * 2 + (g >> 1)];
        wave_lds_fence();
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int p = block * kBlockPos + g * 4 + r, kh = (c & 1) * 4, vh = (g & 1) * 4 + r;
            if (p < span.first || p >= end) continue;
            const float ks = key_scale(pairs[n][r]), vs = value_scale(pairs[n][r]);
            const size_t at = (size_t)(span.row0 + p - span.first) * row_stride + (size_t)head * D +
                              n * kSpan + c * 4;
            const uint32_t a = keys[n][r];
            once_store(k + at, make_float4(nibble(a, kh) * ks, nibble(a, kh + 1) * ks,
                                           nibble(a, kh + 2) * ks, nibble(a, kh + 3) * ks));
            once_store(v + at, make_float4(nibble(w[0], vh) * vs, nibble(w[1], vh) * vs,
                                           nibble(w[2], vh) * vs, nibble(w[3], vh) * vs));
        }
    }
}

// ----------------------------------------------------------------- attention

// One row a stream multiplies on v_mfma_i32_16x16x64_i8. A byte of the cache gives two
// of its operand's by a shift and two ANDs: a number in the upper half of a byte is 16
// times itself as a signed byte. A query (and 64 keys' weights) becomes a fixed-point
// number of 30 bits, split into four signed bytes that stand in four rows of the other
// operand: products and sums are exact, and
//   ((b3 * 2^8 + b2) * 2^16 + (b1 * 2^8 + b0)) * step
// is rounded to fp32.

// Sixteen numbers of the cache -> an operand, 16 times each.
__device__ inline i32x4 unpack16(u32x2 x) {
    return i32x4{(int)(x[0] << 4 & 0xF0F0F0F0u), (int)(x[0] & 0xF0F0F0F0u),
                 (int)(x[1] << 4 & 0xF0F0F0F0u), (int)(x[1] & 0xF0F0F0F0u)};
}
// Bytes of the cache for one row a stream, read once: past the caches.
__device__ inline u32x2 stream_load8(const uint8_t *p) {
    return __builtin_nontemporal_load((const u32x2 *)p);
}

template <int E>
__device__ inline int row_turn(int v) {  // lane i of 16 gets lane (i + E) % 16's
    return __builtin_amdgcn_update_dpp(0, v, 0x120 + 16 - E, 0xf, 0xf, false);
}

struct Kv4Decode {
    const float *q;
    size_t q_stride;
    int group;
    float scale;  // of the scores, times log2 e
    int max_positions, splits, steps;  // a split: steps * W * 64 keys
    // Slot (s * query heads + head) * splits + split.
    float *part_acc, *part_ml;
    float *out;  // splits = 1: the rows themselves (else NULL)
    size_t out_stride;
    // With sums:
    // [streams][query heads]: a weight is 2^(score - top) * share; top is infinite where the
    // row did not come out finite. One number, the logarithm of the sum, would be rounded in
    // units of the score.
    float *tops, *shares;
    float *scores;  // [streams][query heads][max_positions], in units of log 2
    const float *before;
    float *after;  // NULL: another launch adds the weights up
    size_t stride;
};

// A row's top and share, from its sum of weights in units of 2^m: the top is near the sum's
// logarithm, so that the share is near 1 (or m, where that is too large to be added to).
// (The reciprocal is off by one step.)
__device__ inline float2 kv4_share(float m, float total) {
    const bool fine = total > 0.0f && total < INFINITY && fabsf(m) < INFINITY;
    const float top = m + (float)__builtin_amdgcn_frexp_expf(total);
    return make_float2(fine ? top : INFINITY, __builtin_amdgcn_exp2f(top - m) * __builtin_amdgcn_rcpf(total));
}

template <int D, int W, int Q>
struct Kv4DecodeShared {
    __align__(16) uint32_t digits[Q == 1 ? 1 : W][16][16];  // [row][block, quad of keys]
    float acc[W][Q][D];
    float m[W][Q], l[W][Q], top[Q], share[Q];
};

// The exponent of a power of two above |x|; 0 for 0 and for what is not finite.
__device__ inline float exponent_of(float x) { return (float)__builtin_amdgcn_frexp_expf(x); }
// Scores from which on the exponent of a value scale could be lost in a sum with them; what
// stands for all that are larger, and for no key.
constexpr int kVast = 1 << 20;
constexpr float kMostBound = 0x1p30f;

// The largest of 16 lanes, and over those 16 and 32 apart. Of whole numbers: a maximum of
// floats takes four instructions for each lane moved, to quiet NaN, of these one.
__device__ inline int row16_most(int v) {
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0x124, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, true));
    return max(v, __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, true));
}
__device__ inline int xor16_32_most(int v) {
    const auto a = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    v = max((int)a[0], (int)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    return max((int)b[0], (int)b[1]);
}

// One row a stream. A work-group of W waves takes a split's keys of one (stream, key
// head) for Q (1 or 4) of its queries, W * 64 keys a step: a wave's 64 are 4 blocks,
// whose bytes it requests together, the next step's as soon as the registers are free:
// keys after the scores, values after their product. No wave waits for another before
// the joint of all W.
//
// Weights enter their product times their keys' value scales, below 2^m: m is a whole
// number, the largest of score + exponent of the value scale so far, so that one fixed
// point serves the running sums, which stay whole numbers as long as m does. Each 64 dims
// have theirs: a span of small values keeps its bits beside one of large ones. Where scores
// pass 2^20 their sum with an exponent would round it away: scores and m are then counted
// from the largest score so far, whose differences to it are exact.
//
// A lone query's digits stand in rows 4 t .. 4 t + 3 for block t, zeros elsewhere, so
// that lane (g, i) gets the score of key i of block g: one key to a lane. Of four
// queries, lane (g, i) has query g's score of key i of each block.
//
// Bound by the cache's bytes where contexts are long: 256 streams of up to 8187 keys, 567
// MB in 93 us, 6.1 TB/s (a plain read reaches 6.5). Else by the chain of a few steps: 64
// of up to 2048 9.4 us (34 MB; with the scores stored and added up 13.6), one key 3.7, a
// launch. Heads of 128 with 4 queries, 48 streams of up to 4096: 105 MB in 25 us, 24 where
// both halves of a head share m. Vast scores: 64 of up to 2048 11.6.
template <int D, int W, int Q, bool SCORES>
__global__ __launch_bounds__(64 * W, D == 64 ? 5 : Q == 1 ? 4 : 3) void k_kv4_decode(
    Kv4 kv, Kv4Rows rows, Kv4Decode a, int *status) {
    constexpr int N = D / kSpan, T = D / 16, S = Q == 1 ? 1 : 4, A = Q == 1 ? N : T;
    __shared__ Kv4DecodeShared<D, W, Q> sh;
    // Heads vary fastest: with 8 of them a head's passes stay on one XCD.
    const int head = blockIdx.x % kv.heads, j0 = blockIdx.x / kv.heads * Q;
    // The splits in turn by stream: the first ones, which all contexts have, would else be
    // dispatched to the same CUs where their number divides 32.
    const int s = blockIdx.z, split = (blockIdx.y + s) % gridDim.y;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int i = lane & 15, g = lane >> 4;
    int b0 = (split * a.steps * W + wave) * 4;  // the wave's blocks: b0 .. b0 + 3
    const int32_t *table = rows.tables + (size_t)s * rows.table_stride;
    int ids[4];
#pragma unroll
    for (int t = 0; t < 4; t++) ids[t] = uniform_load(table + min(b0 + t, rows.table_stride - 1));
    const Kv4Span span = kv4_span(rows, s, a.max_positions,
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
    const int held = p / kBlockPos + 1;
    const size_t qh0 = (size_t)s * kv.heads * a.group + (size_t)head * a.group + j0;

    const uint8_t *values_of = kv.values + head * (D * kBlockPos);
    const uint32_t *scales_of = kv.scales + head * (N * kBlockPos);
    const unsigned values_step = kv.heads * (D * kBlockPos), scales_step = kv.heads * (N * kBlockPos);
    const unsigned key_at = i * 32 + g * 8, pair_at = i, value_at = N * kPlane + i * 8;
    u32x2 kr[4][N], vr[T];
    uint32_t pair[S][N];
    bool wild = false;
    unsigned on = 0, ever = 0;  // bit t: block t of the step whose keys were requested counts
    // Blocks b .. b + 3; block 0 for one past the last or not in the cache, so that every
    // step requests alike and waits for no more than it needs.
    auto load = [&](int b, bool values) {
        unsigned id[4];
        if (!values) on = 0;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const bool there = b + t < held, in = (unsigned)ids[t] < kv.blocks;
            id[t] = (unsigned)__builtin_amdgcn_readfirstlane(there && in ? ids[t] : 0);
            if (!values) {
                wild |= there && !in;
                on |= (there && in ? 1u : 0u) << t;
            }
        }
        const unsigned mine = g < 2 ? (g ? id[1] : id[0]) : (g == 2 ? id[2] : id[3]);
        if (!values) {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const uint8_t *tile = values_of + (size_t)id[t] * values_step;
#pragma unroll
                for (int n = 0; n < N; n++) kr[t][n] = stream_load8(tile + (key_at + n * kPlane));
            }
#pragma unroll
            for (int t = 0; t < S; t++) {
                const uint32_t *pairs = scales_of + (size_t)(Q == 1 ? mine : id[t]) * scales_step;
#pragma unroll
                for (int n = 0; n < N; n++)
                    pair[t][n] = __builtin_nontemporal_load(pairs + (pair_at + n * kBlockPos));
            }
        } else {
            const uint8_t *tile = values_of + (size_t)mine * values_step + value_at;
#pragma unroll
            for (int t = 0; t < T; t++) vr[t] = stream_load8(tile + t * 128);
        }
    };

    // Row i of the operand: byte i % 4 of query j0 + i / 4.
    const float *q = a.q + (size_t)s * a.q_stride +
                     ((size_t)head * a.group + min(j0 + (Q == 1 ? 0 : i >> 2), a.group - 1)) * D;
    const uint32_t byte = row_byte(i & 3), sel = byte | (4u + byte) << 8;
    i32x4 qd[S == 1 ? 4 : 1][N];
    float step, top = 0.0f;
    auto begin = [&] {
        float4 x[N][4];
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) x[n][k] = *(const float4 *)(q + n * kSpan + g * 16 + k * 4);
        // The order of the requests is the order in which they are waited for.
        __builtin_amdgcn_sched_barrier(0);
        load(b0, false);
        __builtin_amdgcn_sched_barrier(0);
        load(b0, true);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float4 v = x[n][k];
                top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)),
                                       fmaxf(fabsf(v.z), fabsf(v.w))));
                if (!(v.x == v.x && v.y == v.y && v.z == v.z && v.w == v.w)) top = INFINITY;
            }
        top = xor16_32_max(top);
        const int e = fix_exponent(top);
        const float mul = power_of_2(e);
#pragma unroll
        for (int n = 0; n < N; n++) {
            i32x4 d;
#pragma unroll
            for (int k = 0; k < 4; k++)
                d[k] = (int)pick4(fix_bytes(x[n][k].x, mul), fix_bytes(x[n][k].y, mul),
                                  fix_bytes(x[n][k].z, mul), fix_bytes(x[n][k].w, mul), sel);
            if constexpr (Q == 1)
#pragma unroll
                for (int t = 0; t < 4; t++) qd[t][n] = i >> 2 == t ? d : i32x4{0, 0, 0, 0};
            else
                qd[0][n] = d;
        }
        // Fixed point cannot say that a query is infinite. (16: the cache's numbers.)
        step = top < INFINITY ? a.scale * power_of_2(-e) * 0.0625f : __builtin_nanf("");
        if (Q != 1) step = __shfl(step, g * 4);  // of query j0 + g
    };
    // l counts in units of 2^m[0], the sums of 64 dims n in units of 2^m[n].
    float m[N], l = 0.0f, acc[A];
#pragma unroll
    for (int n = 0; n < N; n++) m[n] = -kMostBound;
    float zero = 0.0f;  // the score that m counts from, where scores are vast
    bool vast = false;
    // Whole sums of the values, times 2^34 in their units: of dims 16 t + i, or 64 t + lane. A step
    // adds 2^20 at most, and a work-group has 16 steps at most.
    i32x4 sum[A];
#pragma unroll
    for (int t = 0; t < A; t++) acc[t] = 0.0f, sum[t] = i32x4{0, 0, 0, 0};
    auto flush = [&](const float (&less)[N]) {
#pragma unroll
        for (int t = 0; t < A; t++) {
            const float whole = fmaf((float)sum[t].x, 0x1p24f, fmaf((float)sum[t].y, 0x1p16f,
                                     fmaf((float)sum[t].z, 0x1p8f, (float)sum[t].w)));
            acc[t] = fmaf(whole, 0x1p-34f, acc[t]) * less[t * N / A];
            sum[t] = i32x4{0, 0, 0, 0};
        }
    };

    auto attend = [&](bool more) {
        const unsigned count = on;
        ever |= on;
        if (more)
#pragma unroll
            for (int t = 0; t < 4; t++)
                ids[t] = uniform_load(table + min(b0 + 4 * W + t, rows.table_stride - 1));
        // Scores, in units of log 2.
        float w[S], vs[S][N];
        i32x4 c[S][N];
#pragma unroll
        for (int t = 0; t < S; t++)
#pragma unroll
            for (int n = 0; n < N; n++) c[t][n] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int n = 0; n < N; n++) {
                i32x4 &to = c[Q == 1 ? 0 : t][n];
                to = __builtin_amdgcn_mfma_i32_16x16x64_i8(qd[Q == 1 ? t : 0][n], unpack16(kr[t][n]),
                                                           to, 0, 0, 0);
            }
#pragma unroll
        for (int t = 0; t < S; t++) {
            const int b = b0 + (Q == 1 ? g : t);
            const bool seen = (count >> (Q == 1 ? g : t) & 1) && b * kBlockPos + i <= p;
            float score = 0.0f;
#pragma unroll
            for (int n = 0; n < N; n++) {
                score = fmaf(fix_sum(c[t][n]), key_scale(pair[t][n]), score);
                vs[t][n] = seen ? value_scale(pair[t][n]) : 0.0f;
            }
            w[t] = seen ? score * step : -INFINITY;
            if (SCORES && b * kBlockPos + i <= p && (Q == 1 || g < live))
                a.scores[(qh0 + (Q == 1 ? 0 : g)) * a.max_positions + b * kBlockPos + i] = w[t];
        }
        // Whole numbers that no score + exponent of a value scale passes.
        int bound[N];
#pragma unroll
        for (int n = 0; n < N; n++) {
            float b = -kMostBound;
#pragma unroll
            for (int t = 0; t < S; t++) b = fmaxf(b, w[t] + exponent_of(vs[t][n]));
            bound[n] = row16_most((int)ceilf(fminf(b, kMostBound)));
            if (Q == 1) bound[n] = xor16_32_most(bound[n]);
        }
        if (more) load(b0 + 4 * W, false);
        float next[N], best = kNone;
        const bool before = vast;
#pragma unroll
        for (int n = 0; n < N; n++) next[n] = fmaxf(m[n], (float)bound[n]);
        if (vast || __any(abs(bound[0]) >= kVast)) {
#pragma unroll
            for (int t = 0; t < S; t++) best = fmaxf(best, w[t]);
            best = row16_max(best);
            if (Q == 1) best = xor16_32_max(best);
            best = ceilf(best);
            vast |= __any(best > kNone && abs(bound[0]) >= kVast);
        }
        if (vast) {
            const bool none = m[0] <= -kMostBound;  // no key so far
            const float last = before || none ? zero : m[0], from = before ? 0.0f : last;
            zero = none ? best : fmaxf(last, best);
#pragma unroll
            for (int t = 0; t < S; t++) w[t] -= zero;
#pragma unroll
            for (int n = 0; n < N; n++) {
                if (!none) m[n] = m[n] - from - (zero - last);
                float b = kNone;
#pragma unroll
                for (int t = 0; t < S; t++) b = fmaxf(b, w[t] + exponent_of(vs[t][n]));
                b = row16_max(b);
                if (Q == 1) b = xor16_32_max(b);
                next[n] = fmaxf(m[n], ceilf(b));
            }
        }
        bool grows = false;
#pragma unroll
        for (int n = 0; n < N; n++) grows |= next[n] != m[n];
        if (__any(grows)) {
            float less[N];
#pragma unroll
            for (int n = 0; n < N; n++) {
                less[n] = __builtin_amdgcn_exp2f(m[n] - next[n]);  // no key so far: 0
                m[n] = next[n];
            }
            flush(less);
            l *= less[0];
        }
#pragma unroll
        for (int t = 0; t < S; t++) {
            w[t] = __builtin_amdgcn_exp2f(w[t] - m[0]);
            l += w[t];
        }
#pragma unroll
        for (int n = 0; n < N; n++) {
            const float fix = n ? __builtin_amdgcn_exp2f(m[0] - m[n]) * 0x1p30f : 0x1p30f;
            if constexpr (Q == 1) {
                // Digit t of block g's keys, a quad of keys a word, in row t of dims 16 j ..
                // 16 j + 15, which are rows 4 j .. 4 j + 3: their first word is quad j's.
                const uint32_t u = fix_bytes(w[0] * vs[0][n], fix);
                const int word = (int)pick4(quad_lane<0>(u), quad_lane<1>(u), quad_lane<2>(u),
                                            quad_lane<3>(u), sel);
                const i32x4 turned = {word, row_turn<4>(word), row_turn<8>(word), row_turn<12>(word)};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const i32x4 x = unpack16(vr[n * 4 + j]);
                    sum[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                        i >> 2 == j ? turned : i32x4{0, 0, 0, 0},
                        i32x4{x[j], x[(j + 1) & 3], x[(j + 2) & 3], x[(j + 3) & 3]}, sum[n], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const uint32_t u = fix_bytes(w[t] * vs[t][n], fix);
                    sh.digits[wave][g * 4 + (i & 3)][t * 4 + (i >> 2)] =
                        pick4(quad_lane<0>(u), quad_lane<1>(u), quad_lane<2>(u), quad_lane<3>(u), sel);
                }
                wave_lds_fence();
                const i32x4 pd = *(const i32x4 *)&sh.digits[wave][i][g * 4];
                wave_lds_fence();
#pragma unroll
                for (int t = n * 4; t < n * 4 + 4; t++)
                    sum[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(pd, unpack16(vr[t]), sum[t], 0, 0, 0);
            }
        }
        b0 += 4 * W;
        if (more) load(b0, true);
    };
    // The last step apart: no branch stands between a request and its wait.
    int steps = b0 < held ? min(a.steps, (held - b0 - 1) / (4 * W) + 1) : 0;
    if (steps > 0) {
        begin();
        for (; steps > 1; steps--) attend(true);
        attend(false);
        // All in units of 2^m[0]; where scores are vast, whose m is an exponent below 2^6, of
        // 2^zero.
        float unit[N];
#pragma unroll
        for (int n = 0; n < N; n++)
            unit[n] = n || vast ? __builtin_amdgcn_exp2f(vast ? m[n] : m[n] - m[0]) : 1.0f;
        flush(unit);
        l *= unit[0];
        if (m[0] <= -kMostBound) m[0] = kNone;
        if (vast) m[0] = zero;
    }
    if (wild && lane == 0) atomicOr(status, 2);
    l = row16_sum(l);
    if (Q == 1) l = xor16_32_sum(l);
#pragma unroll
    for (int t = 0; t < A; t++) sh.acc[wave][Q == 1 ? 0 : g][Q == 1 ? t * 64 + lane : t * 16 + i] = acc[t];
    if (g < Q && i == 0) {
        sh.m[wave][g] = ever ? m[0] : -INFINITY;
        sh.l[wave][g] = l;
    }
    bool bad = !(top < INFINITY);
    // What U keys weighed before, on its way while the waves are joined.
    constexpr int U = 8;
    const size_t sums_at = ((size_t)s * kv.heads + head) * a.stride;
    float weighed[U];
    auto load_weighed = [&](int from) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int e = from + u * 64 * W;
            weighed[u] = a.before && e < p ? a.before[sums_at + e] : 0.0f;
        }
    };
    if (SCORES && a.after) load_weighed(threadIdx.x);
    __syncthreads();
    for (int e = threadIdx.x; e < live * D; e += 64 * W) {
        const int j = e / D, d = e % D;
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < W; n++) mx = fmaxf(mx, sh.m[n][j]);
        float total = 0.0f, o = 0.0f;
#pragma unroll
        for (int n = 0; n < W; n++) {
            // A wave without a key: m = -inf, l = 0, acc = 0.
            const float c = __builtin_amdgcn_exp2f(sh.m[n][j] - fmaxf(mx, kNone));
            total = fmaf(sh.l[n][j], c, total);
            o = fmaf(sh.acc[n][j][d], c, o);
        }
        if (a.out) {
            // Scores that are all -inf: not finite. No key: zeros.
            o = mx == -INFINITY ? 0.0f : o / total;
            a.out[(size_t)s * a.out_stride + ((size_t)head * a.group + j0 + j) * D + d] = o;
            if (SCORES && d == 0) {
                const float2 x = kv4_share(mx, total);
                a.tops[qh0 + j] = sh.top[j] = x.x;
                a.shares[qh0 + j] = sh.share[j] = x.y;
            }
            bad |= !isfinite(o);
        } else {
            const size_t at = (qh0 + j) * a.splits + split;
            a.part_acc[at * D + d] = o;
            if (d == 0) *(float2 *)(a.part_ml + at * 2) = make_float2(mx, total);
        }
    }
    flag_nonfinite(status, bad);
    if (!SCORES || !a.after) return;
    __syncthreads();
    for (int e0 = threadIdx.x; e0 <= p; e0 += 64 * W * U) {
        float part[U][Q];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < Q; j++) {
                const int e = e0 + u * 64 * W;
                part[u][j] = j < live && e <= p ? a.scores[(qh0 + j) * a.max_positions + e] : -INFINITY;
            }
        if (e0 > (int)threadIdx.x) load_weighed(e0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int e = e0 + u * 64 * W;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < Q; j++)
                if (j < live && sh.top[j] < INFINITY)
                    sum = fmaf(__builtin_amdgcn_exp2f(part[u][j] - sh.top[j]), sh.share[j], sum);
            if (e <= p) a.after[sums_at + e] = weighed[u] + sum;
        }
    }
}

// Where a tile of 16 rows and a query head stand among rows + 16 * streams rows.
__device__ inline size_t tile_at(const Kv4Span &span, int s, int r0, int qh, int wide) {
    return (size_t)(span.row0 + 16 * s + r0) * wide + (size_t)qh * 16;
}

constexpr float kMostFused = 0x1p23f;  // of scores that are not vast
constexpr uint32_t kExponent = 0x7F800000, kVastRow = 0x80000000;

// A run's row as its sums read it: a weight is 2^(score - top) * share, from its sum of
// weights in units of 2^m. The share, a number in [1/2, 1), stands in the last 23 bits of the
// row's word, whose exponent is that of the scores' factor. A vast row's top is m, and 16 bits
// of the share stand behind 7 of the sum's exponent.
__device__ inline uint32_t kv4_factor(float m, float total, uint32_t factor, float &top) {
    const bool fine = total > 0.0f && total < INFINITY && fabsf(m) < INFINITY;
    const float f = bitsf((fbits(total) & ~kExponent) | 0x3F800000u);  // [1, 2)
    int e = (int)(fbits(total) >> 23) - 127;
    uint32_t share = 0;  // of 1 / 2
    if (f == 1.0f)
        e--;
    else
        share = fbits(1.0f / f) & ~kExponent;
    const bool vast = fabsf(m) >= kMostFused;
    top = fine ? (vast ? m : m + (float)e) : INFINITY;
    return (factor & kExponent) | (vast ? kVastRow | (uint32_t)((e + 64) & 127) << 16 | share >> 7 : share);
}

// The splits of a row's query head joined: D / 4 lanes for 4 dims each, times G that
// share the splits. `keys`: of a split, or 0: every split has its part of every row, or
// says that it has none (a maximum of -inf). Bound by its launch: 4.5 us for 256 streams
// of up to 8 splits, 8 heads of 64; 3.8 for 48 of 4 splits, 32 query heads of 128.
template <int D, int G>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4 kv, Kv4Rows rows, const float *part_acc,
                                                  const float *part_ml, int group,
                                                  int max_positions, int splits, int keys,
                                                  float *out, size_t out_stride, float *tops,
                                                  float *shares, uint32_t *factors,
                                                  int *status) {
    constexpr int L = D / 4, M = L * G;
    const int s = blockIdx.z, wide = kv.heads * group;
    const size_t e = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int lane = (int)(e % M), share = lane / L, d = lane % L * 4;
    const int qh = (int)(e / M % wide);
    const size_t i = e / M / wide;
    const Kv4Span span = kv4_span(rows, s, max_positions, false, status);
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
    const float base = fmaxf(mx, kNone);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < n; j0 += M) {
        const int last = min(M, n - j0);
        const float2 ml = lane < last ? *(const float2 *)(part_ml + (at + j0 + lane) * 2)
                                      : make_float2(-INFINITY, 0.0f);
        const float c = __builtin_amdgcn_exp2f(ml.x - base);
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
    // No key that counts: zeros. Scores that are all -inf: not finite.
    if (mx != -INFINITY) o = make_float4(o.x / total, o.y / total, o.z / total, o.w / total);
    *(float4 *)dst = o;
    if (d == 0 && shares) {
        const float2 x = kv4_share(mx, total);
        tops[row * wide + qh] = x.x;
        shares[row * wide + qh] = x.y;
    } else if (d == 0 && factors) {
        uint32_t &factor = factors[tile_at(span, s, (int)i & ~15, qh, wide) + (i & 15)];
        factor = kv4_factor(mx, total, factor, tops[row * wide + qh]);
    }
    flag_nonfinite(status, !(isfinite(o.x) && isfinite(o.y) && isfinite(o.z) && isfinite(o.w)));
}

// One row a stream's weights, from its scores: a thread for each key of a (stream, key
// head).
__global__ __launch_bounds__(256) void k_kv4_sums_one(Kv4 kv, Kv4Rows rows, Kv4Decode a,
                                                      int *status) {
    const int head = blockIdx.y, s = blockIdx.z, p = blockIdx.x * 256 + threadIdx.x;
    const Kv4Span span = kv4_span(rows, s, a.max_positions, false, status);
    if (!span.live || p > span.first) return;
    const size_t at = ((size_t)s * kv.heads + head) * a.stride + p;
    const size_t qh0 = ((size_t)s * kv.heads + head) * a.group;
    float sum = 0.0f;
    for (int j = 0; j < a.group; j++) {
        const float top = a.tops[qh0 + j], score = a.scores[(qh0 + j) * a.max_positions + p];
        if (top < INFINITY) sum = fmaf(__builtin_amdgcn_exp2f(score - top), a.shares[qh0 + j], sum);
    }
    a.after[at] = (a.before && p < span.first ? a.before[at] : 0.0f) + sum;
}

// Runs of rows: a work-group of 4 waves takes 4 tiles of 16 rows of one query head each
// (the query heads of a key head side by side), and passes over the keys 64 at a time:
// each wave turns one block into fp16 in LDS (number times scale: exact), where all four
// read it, while the next 64 keys' bytes are on their way. Scores are taken keys by rows
// (K Q^T), so that a lane holds 16 of its row's scores and the weights are the next
// product's operand as they stand (O^T = V^T P^T). A query and a weight are two fp16
// terms (22 bits). The running maximum is a whole number (in units of log 2), so that
// rescaling is exact and rare; weights stand 2^14 higher, which keeps their low terms
// normal. A score less the maximum is one multiply-add, which is
// within 1/4 of what the rounded score less the maximum is, up to 2^23; where queries or
// keys are so large that scores can pass that, they are rounded as the maximum is.
//
// So a weight is held to 2^-37 of the row's largest, which serves while value scales are
// alike. A block with one that is not within 2^5 of the first block's is far: its values
// are staged with their scales' exponents made the first block's, and its weights enter
// the product times the difference, 2^shift. The products are then held to the largest
// weight times 2^shift, 2^lift times the largest weight by itself, which the row's sum of
// weights is held to; that is taken in fp32 as long as the two differ. So no row loses
// bits to a key that weighs little but whose values are large, nor the other way round.
// Each 64 dims have a first block's exponent, shifts and a lift of their own.
//
// Bound by vector and matrix instructions, which hardly overlap: for a tile and 64 keys
// about 800 cycles of a SIMD's vector units (256 of them the exponentials) and 576 of its
// matrix cores, 1376 one after the other; it takes about 1750, as waves whose rows are short
// end early. 8187 rows of one prompt, 8 heads of 64: 189 us, 137 GFLOP with the two terms,
// 0.73 PFLOP/s (a library product: 1.3); 295 with every second block far, 193 where queries
// may give vast scores, 227 where keys may. Eight waves that share a block's staging 193 for
// 182; two copies of the loop's body, masked and not, 346 (they spill). 5 prompts of up to
// 1777 rows and 16 query heads 70 us; 3 of up to 300, behind 200, 14.0: up to 8 chunks, one
// after the other.
struct Kv4Run {
    const float *q;
    size_t q_stride;
    int group;
    float scale;  // of the scores, times log2 e
    int max_positions, splits;
    float *part_acc, *part_ml;
    float *out;  // splits = 1: the rows themselves
    size_t out_stride;
    // With sums: the rows' tops, [rows][query heads]; and the last `counted` rows' queries as
    // operands and their words (kv4_factor), tile by tile (tile_at).
    float *tops;
    uint4 *queries;
    uint32_t *factors;
    int counted;
};

template <int D>
struct Kv4RunShared {
    f16x8 k[2][4][D / 32][64];  // [buffer][block][step][lane]
    f16x8 v[2][2][D / 16][64];  // [buffer][pair of blocks][16 dims][lane]
    // [buffer][block][64 dims][key], of far blocks
    __align__(16) float shift[2][4][D / kSpan][kBlockPos];
    // [buffer][block]: bit 0: not in the cache; bit 1: far; bit 2: of large keys
    uint8_t kind[2][4];
    float lift[4][D / kSpan][16];  // [wave][64 dims][row]
};

// Numbers of the cache become fp16 two at a time, numbers b and b + 2 of a word's halves:
// eight in the order 0, 2, 4, 6, 1, 3, 5, 7, four in the order 0, 2, 1, 3, which the other
// operands keep to.
//
// Four in the low halves of bytes, plus 8, times their scales: 0x6400 | n is 1024 + n.
__device__ inline f16x4 halves_f16(uint32_t n, f16x2 s02, f16x2 s13) {
    const f16x2 off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    const uint32_t even = __builtin_amdgcn_perm(0x64646464u, n, 0x04020400u);
    const uint32_t odd = __builtin_amdgcn_perm(0x64646464u, n, 0x04030401u);
    const f16x2 a = (__builtin_bit_cast(f16x2, even) + off) * s02;
    const f16x2 b = (__builtin_bit_cast(f16x2, odd) + off) * s13;
    return f16x4{a.x, a.y, b.x, b.y};
}
__device__ inline f16x8 word_f16(uint32_t w, f16x2 s2) {
    const uint32_t u = w ^ 0x88888888u;
    return __builtin_shufflevector(halves_f16(u & 0x0F0F0F0Fu, s2, s2),
                                   halves_f16(u >> 4 & 0x0F0F0F0Fu, s2, s2), 0, 1, 4, 5, 2, 3, 6, 7);
}
// The same in one multiply-add: a number plus 8 in bits 6 .. 9 (and 22 .. 25) of `shifted`
// is 1 + n / 16 with an exponent before it; times 16 s, less 24 s, which is exact, as
// long as 24 s is an fp16 number.
constexpr uint16_t kMostFast = 0x6950;  // 2720
// Key scales up to 64 are ordinary: a score is less than the query's largest element, 2^15,
// times 8 * 64 in each dim.
constexpr uint16_t kOrdinary = 0x5400;
struct PairBits {
    uint32_t mask = 0x03C003C0u, one = 0x3C003C00u;
    // In registers: an AND-OR takes no literals.
    __device__ PairBits() { asm("" : "+s"(mask), "+v"(one)); }
};
__device__ inline f16x2 pair_f16(uint32_t shifted, f16x2 s16, f16x2 s24, const PairBits &b) {
    return __builtin_elementwise_fma(
        __builtin_bit_cast(f16x2, (shifted & b.mask) | b.one), s16, -s24);
}
__device__ inline f16x2 times(f16x2 s, float f) { return s * f16x2{(_Float16)f, (_Float16)f}; }

// A wave's queries -> two fp16 terms of 64 dims a step pair, scaled to a largest element
// in [2^14, 2^15), and the factor of the scores. x: [64 dims][quarter] of dims 16 g on.
template <int D>
__device__ inline float kv4_query(const float4 (&x)[D / kSpan][4], float scale, float &biggest,
                                  f16x8 (&hi)[D / 32], f16x8 (&lo)[D / 32]) {
    biggest = 0.0f;
#pragma unroll
    for (int n = 0; n < D / kSpan; n++)
#pragma unroll
        for (int k = 0; k < 4; k++)
            biggest = fmaxf(biggest, fmaxf(fmaxf(fabsf(x[n][k].x), fabsf(x[n][k].y)),
                                           fmaxf(fabsf(x[n][k].z), fabsf(x[n][k].w))));
    biggest = xor16_32_max(biggest);
    const int e = min(126, 141 - (int)(fbits(biggest) >> 23));
    // The factor of the scores stays above 0, for a scale of 0 too.
    const float mul = scale == 0.0f ? 0.0f : copysignf(power_of_2(e), scale);
#pragma unroll
    for (int n = 0; n < D / kSpan; n++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
            f16x2 h[4], o[4];
#pragma unroll
            for (int z = 0; z < 2; z++) {
                const float4 v = x[n][k * 2 + z];
                split_pair(v.x * mul, v.z * mul, h[z], o[z]);
                split_pair(v.y * mul, v.w * mul, h[z + 2], o[z + 2]);
            }
            hi[n * 2 + k] = join_pairs(h[0], h[1], h[2], h[3]);
            lo[n * 2 + k] = join_pairs(o[0], o[1], o[2], o[3]);
        }
    return scale == 0.0f ? 1.0f : fmaxf(fabsf(scale) * power_of_2(-e), 0x1p-126f);
}

// NaN if one is NaN. (No asm: what it reads may come from a matrix instruction.)
__device__ inline float largest(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

template <int D>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void k_kv4_run(Kv4 kv, Kv4Rows rows, Kv4Run a,
                                                                  int *status) {
    constexpr int N = D / kSpan, KS = D / 32, T = D / 16;
    __shared__ Kv4RunShared<D> sh;
    // Heads fastest (with 8 of them a head's keys stay in one XCD's L2), the longest rows
    // first, and every second 256 work-groups the other way round: a CU, which gets each
    // 256th, has long and short ones.
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
    const Kv4Span span = kv4_span(rows, s, a.max_positions,
                                  threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0, status);
    const int tiles = (span.count + 15) / 16 * a.group;
    if (bx * 4 >= tiles) return;
    const int tile = bx * 4 + wave, r0 = tile / a.group * 16;
    const int qh = head * a.group + tile % a.group, wide = kv.heads * a.group;
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
    // Keys to be seen by some row here. Splits take the chunks of 64 in turn, so that each
    // has its share of every row's.
    const int keys = span.first +
                     min(span.count, (min(bx * 4 + 3, tiles - 1) / a.group + 1) * 16);
    const int c0 = split, stride = a.splits, c1 = (keys + 63) / 64;
    const int p0 = span.first + r0;
    int p = i < live ? p0 + i : -1;  // this lane's row
    asm("" : "+v"(p));  // else p0 + i takes a register of its own throughout
    const int wave_top = p0 + live - 1;

    const float *q = a.q + row * a.q_stride + (size_t)qh * D;
    f16x8 qhi[KS], qlo[KS];
    float qs, biggest;
    {
        float4 x[N][4];
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) x[n][k] = *(const float4 *)(q + n * kSpan + g * 16 + k * 4);
        qs = kv4_query<D>(x, a.scale, biggest, qhi, qlo);
    }
    if (a.queries && split == 0 && live > 0 && r0 + 16 > span.count - a.counted) {
        const size_t at = tile_at(span, s, r0, qh, wide);
        uint4 *to = a.queries + at * (D / 4) + lane;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            to[k * 128] = __builtin_bit_cast(uint4, qhi[k]);
            to[k * 128 + 64] = __builtin_bit_cast(uint4, qlo[k]);
        }
        if (g == 0) a.factors[at + i] = fbits(qs) & kExponent;
    }

    // Chunk c: its bytes requested, then turned into LDS; wave w takes block w. The block's
    // id of the j-th chunk waits in lane j (j below 64, then the next 64): no chunk waits
    // for its own. Lane (g, i): 16 dims of key i; keys 4 g .. 4 g + 3 of dims 16 t + i.
    const unsigned key_at = i * 32 + g * 8, value_at = N * kPlane + i * 8 + (g >> 1) * 4;
    const unsigned scale_at = i, scales_at = g * 4;
    u32x2 kr[N];
    uint32_t vr[T], ks[N];
    u32x4 vs[N];
    int raw_of = 0, raw = 0;
    bool wild = false;
    const int32_t *table = rows.tables + (size_t)s * rows.table_stride;
    const int end = span.first + span.count;
    // The exponents of the first block's largest value scales.
    constexpr int kNear = 5;
    auto exponent = [](float x) { return max((int)(fbits(x) >> 23) - 127, -17); };
    int usual[N];
    uint32_t least_near[N], range_near[N];  // scale pairs that are not far
    auto look_first = [&] {
        const int front = table[c0 * 4];
        const uint32_t *sc = kv4_scales<D>(kv, (unsigned)front < kv.blocks ? front : 0, head);
#pragma unroll
        for (int n = 0; n < N; n++) {
            const float x = value_scale(sc[n * kBlockPos + i]);
            const bool in = c0 * 64 + i < end && x >= kLeastScale && x <= kMostScale;
            usual[n] = __builtin_amdgcn_readfirstlane(exponent(row16_max(in ? x : kLeastScale)));
            const uint16_t least = __builtin_bit_cast(uint16_t, (_Float16)power_of_2(max(usual[n] - kNear, -17)));
            const uint16_t past = __builtin_bit_cast(uint16_t, (_Float16)power_of_2(min(usual[n] + kNear + 1, 15)));
            least_near[n] = (uint32_t)least << 16;
            range_near[n] = ((uint32_t)min(past, kMostFast) << 16) - least_near[n];
        }
    };
    auto request = [&](int c, int nth) {
        const int j = nth & 63;
        if (j == 0) {
            const int at = c + lane * stride, b = at * 4 + wave;
            // Past the keys: block 0's bytes, for keys that no row sees.
            raw_of = at < c1 && b * kBlockPos < keys ? table[b] : 0;
            wild |= (unsigned)raw_of >= kv.blocks;
        }
        raw = __builtin_amdgcn_readlane(raw_of, j);
        const unsigned id = (unsigned)raw < kv.blocks ? (unsigned)raw : 0u;
        const uint8_t *tl = kv4_tile<D>(kv, id, head);
        const uint32_t *sc = kv4_scales<D>(kv, id, head);
#pragma unroll
        for (int n = 0; n < N; n++) {
            kr[n] = *(const u32x2 *)(tl + (key_at + n * kPlane));
            ks[n] = sc[scale_at + n * kBlockPos];
            vs[n] = *(const u32x4 *)(sc + (scales_at + n * kBlockPos));
#pragma unroll
            for (int t = 0; t < 4; t++)
                vr[n * 4 + t] = *(const uint32_t *)(tl + (value_at + n * kPlane + t * 128));
        }
    };
    auto stage = [&](int buf, int c) {
        // Most blocks are full, and have value scales that are not far and key scales of
        // ordinary size. Scales order like their bits.
        bool odd = false;
#pragma unroll
        for (int n = 0; n < N; n++)
            odd |= ks[n] - least_near[n] >= range_near[n] || (uint16_t)ks[n] > kOrdinary;
        odd = c * 64 + wave * 16 + 16 > end || __any(odd);
        uint32_t kind = (unsigned)raw >= kv.blocks ? 1 : 0;
        if (!odd) {
            const PairBits bits;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const f16x2 s2 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(ks[n], ks[n], 0x01000100u));
                const f16x2 k16 = times(s2, 16.0f), k24 = times(s2, 24.0f);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const uint32_t u = kr[n][k] ^ 0x88888888u;
                    sh.k[buf][wave][n * 2 + k][lane] =
                        join_pairs(pair_f16(u << 6, k16, k24, bits), pair_f16(u << 2, k16, k24, bits),
                                   pair_f16(u >> 2, k16, k24, bits), pair_f16(u >> 6, k16, k24, bits));
                }
                const f16x2 s02 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(vs[n][2], vs[n][0], 0x07060302u));
                const f16x2 s13 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(vs[n][3], vs[n][1], 0x07060302u));
                const f16x2 a16 = times(s02, 16.0f), a24 = times(s02, 24.0f);
                const f16x2 b16 = times(s13, 16.0f), b24 = times(s13, 24.0f);
                const int left = g & 1 ? 2 : 6, right = g & 1 ? 6 : 2;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const uint32_t u = vr[n * 4 + t] ^ 0x88888888u;
                    const f16x2 a = pair_f16(u << left, a16, a24, bits),
                                b = pair_f16(u >> right, b16, b24, bits);
                    *((f16x4 *)&sh.v[buf][wave >> 1][n * 4 + t][lane] + (wave & 1)) =
                        f16x4{a.x, a.y, b.x, b.y};
                }
            }
        } else {
            // Rows that nothing was written to, or that were not finite, are not far.
            const bool held = c * 64 + wave * 16 + i < end;
            bool far = false, large = false;
#pragma unroll
            for (int n = 0; n < N; n++) {
                large |= held && (uint16_t)ks[n] > kOrdinary && (uint16_t)ks[n] < 0x7C00;
                far |= held && ks[n] < 0x7C000000u && ks[n] - least_near[n] >= range_near[n];
            }
            far = __any(far);
            if (far) kind |= 2;
            if (__any(large)) kind |= 4;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const f16x2 s2 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(ks[n], ks[n], 0x01000100u));
#pragma unroll
                for (int k = 0; k < 2; k++) sh.k[buf][wave][n * 2 + k][lane] = word_f16(kr[n][k], s2);
                // Their values stay finite (the key's scale says if they were not): no
                // weight of theirs reaches a sum.
                float x[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    x[r] = value_scale(vs[n][r]);
                    if (!(x[r] <= kMostScale) || x[r] < 0.0f) x[r] = 0.0f;
                    if (far) {
                        const int shift = x[r] >= kLeastScale ? exponent(x[r]) - usual[n] : 0;
                        x[r] = ldexpf(x[r], -shift);
                        if (i == 0) sh.shift[buf][wave][n][g * 4 + r] = (float)shift;
                    }
                }
                const f16x2 s02 = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x[0], x[2]));
                const f16x2 s13 = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x[1], x[3]));
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const uint32_t u = (vr[n * 4 + t] >> (g & 1) * 4 & 0x0F0F0F0Fu) ^ 0x08080808u;
                    *((f16x4 *)&sh.v[buf][wave >> 1][n * 4 + t][lane] + (wave & 1)) =
                        halves_f16(u, s02, s13);
                }
            }
        }
        if (lane == 0) sh.kind[buf][wave] = (uint8_t)kind;
    };

    // The weights' sums: the row's, taken with the values on the matrix cores (all elements
    // are the same); where blocks are far, or a row is lifted (apart), of this lane's keys on
    // the vector units.
    float m = kNone, l = 0.0f;
    bool apart = false;
    // Queries so large that scores of keys of ordinary size can be vast.
    const bool hot = __any(qs * (D * 0x1p24f) >= kMostFused && biggest < INFINITY);
    f32x4 acc[T], total = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < T; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto attend = [&](int buf, int c, bool masked) {
        const uint32_t kind = (uint32_t)__builtin_amdgcn_readfirstlane(*(const int *)sh.kind[buf]);
        f32x4 w[4];
        // The last key that this lane's row sees, from its own first one on.
        const int last = p - c * 64 - g * 4;
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
        const bool lifts = (kind & 0x02020202u) != 0 || apart;
        auto shifts = [&](int t, int n) {
            f32x4 z = {0.f, 0.f, 0.f, 0.f};
            if (kind >> (8 * t) & 2) z = *(const f32x4 *)&sh.shift[buf][t][n][g * 4];
            return z;
        };
        float mn;
        auto look = [&] {
            float mx[4];
#pragma unroll
            for (int t = 0; t < 4; t++)
                mx[t] = largest(largest(w[t][0], w[t][1], w[t][2]), w[t][3], w[t][3]);
            const float least =
                ceilf(quarters_max(largest(largest(mx[0], mx[1], mx[2]), mx[3], mx[3])) * qs);
            mn = max3(m, least, least);
        };
        if (kind == 0 && !apart) {
            look();
        } else {
#pragma unroll
            for (int t = 0; t < 4; t++)
                if (kind >> (8 * t) & 1) w[t] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            look();
            if (lifts) {
                bool lifted = false;
#pragma unroll
                for (int n = 0; n < N; n++) {
                    float x = -INFINITY;
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const f32x4 z = shifts(t, n);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const float y = (w[t][r] * qs - mn) + z[r];
                            x = max3(x, y, y);
                        }
                    }
                    const float old = sh.lift[wave][n][i];
                    const float lift = fmaxf(old + (m - mn), ceilf(quarters_max(x)));
                    sh.lift[wave][n][i] = lift;
                    lifted |= lift != 0.0f;
                    if (__any(lift != old)) {
                        const float lower = __builtin_amdgcn_exp2f(old - lift);
#pragma unroll
                        for (int t = n * 4; t < n * 4 + 4; t++)
#pragma unroll
                            for (int r = 0; r < 4; r++) acc[t][r] *= lower;
                    }
                }
                apart = __any(lifted);
            }
        }
        if (__any(mn != m)) {
            const float shrink = __builtin_amdgcn_exp2f(m - mn);
            l *= shrink;
#pragma unroll
            for (int t = 0; t < T; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[t][r] *= shrink;
#pragma unroll
            for (int r = 0; r < 4; r++) total[r] *= shrink;
            m = mn;
        }
        const float base = 14.0f - m;
        if (!(hot || lifts || (kind & 0x04040404u) != 0)) {
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) w[t][r] = __builtin_amdgcn_exp2f(fmaf(w[t][r], qs, base));
        } else {
            const bool vast = fabsf(m) >= kMostFused;
            if (__any(vast))
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (vast) w[t][r] = w[t][r] * qs - m;
            const float f = vast ? 1.0f : qs, b = vast ? 14.0f : base;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) w[t][r] = __builtin_amdgcn_exp2f(fmaf(w[t][r], f, b));
            if (lifts)
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) l += w[t][r];
        }
        f16x8 ph[2], pl[2];
#pragma unroll
        for (int n = 0; n < N; n++) {
            if (lifts) {  // from the last 64 dims' shifts and lift to these
                const float down = sh.lift[wave][n][i] - (n ? sh.lift[wave][n - 1][i] : 0.0f);
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    f32x4 z = shifts(t, n);
                    if (n) z -= shifts(t, n - 1);
#pragma unroll
                    for (int r = 0; r < 4; r++) w[t][r] *= __builtin_amdgcn_exp2f(z[r] - down);
                }
            }
            if (n == 0 || lifts) {
                f16x2 hi[4][2], lo[4][2];
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    split_pair(w[t][0], w[t][2], hi[t][0], lo[t][0]);
                    split_pair(w[t][1], w[t][3], hi[t][1], lo[t][1]);
                }
#pragma unroll
                for (int z = 0; z < 2; z++) {
                    ph[z] = join_pairs(hi[z * 2][0], hi[z * 2][1], hi[z * 2 + 1][0], hi[z * 2 + 1][1]);
                    pl[z] = join_pairs(lo[z * 2][0], lo[z * 2][1], lo[z * 2 + 1][0], lo[z * 2 + 1][1]);
                }
            }
            const int t0 = n * 4;
#pragma unroll
            for (int z = 0; z < 2; z++) {
                f16x8 v[4];
#pragma unroll
                for (int t = 0; t < 4; t++) v[t] = sh.v[buf][z][t0 + t][lane];
                if (n == 0) {
                    const int one = lifts ? 0 : 0x3C003C00;
                    const f16x8 ones = __builtin_bit_cast(f16x8, i32x4{one, one, one, one});
                    total = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph[z], total, 0, 0, 0);
                    total = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[z], total, 0, 0, 0);
                }
#pragma unroll
                for (int t = 0; t < 4; t++)
                    acc[t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[t], ph[z],
                                                                         acc[t0 + t], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < 4; t++)
                    acc[t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[t], pl[z],
                                                                         acc[t0 + t], 0, 0, 0);
            }
        }
    };

    if (c0 < c1) {
        request(c0, 0);
#pragma unroll
        for (int n = 0; n < N; n++) sh.lift[wave][n][i] = 0.0f;
        look_first();
        stage(0, c0);
        __syncthreads();
        for (int c = c0, n = 0; c < c1; c += stride, n++) {
            const int buf = n & 1;
            const bool more = c + stride < c1;
            if (more) request(c + stride, n + 1);
            if (live > 0 && c * 64 <= wave_top)
                attend(buf, c, c * 64 + 63 > p0 || live < 16);
            if (more) stage(buf ^ 1, c + stride);
            __syncthreads();
        }
    }
    if (__any(wild) && lane == 0) atomicOr(status, 2);
    l = xor16_32_sum(l) + total[0];
    bool bad = false;
    if (i < live) {
        float base = m;
        if (l == 0.0f) {
            // No key of this split counts (zeros), or all scores are -inf (not finite).
            bool any = false;
            for (int c = c0; c * 64 <= p; c += stride)
                for (int b = c * 4; b < c * 4 + 4 && b * kBlockPos <= p; b++)
                    any |= (unsigned)table[b] < kv.blocks;
            if (!any) base = -INFINITY;
        }
        const size_t at = (((size_t)s * rows.max_rows + r0 + i) * wide + qh) * a.splits + split;
        float *dst = a.splits == 1 ? a.out + row * a.out_stride + (size_t)qh * D : a.part_acc + at * D;
        float f[N];
#pragma unroll
        for (int n = 0; n < N; n++) {
            const float unit = apart ? __builtin_amdgcn_exp2f(sh.lift[wave][n][i]) : 1.0f;
            f[n] = a.splits > 1 ? unit * 0x1p-14f : base == -INFINITY ? 0.0f : unit / l;
        }
#pragma unroll
        for (int t = 0; t < T; t++) {
            const float4 o = make_float4(acc[t][0] * f[t / 4], acc[t][1] * f[t / 4], acc[t][2] * f[t / 4],
                                         acc[t][3] * f[t / 4]);
            bad |= !(isfinite(o.x) && isfinite(o.y) && isfinite(o.z) && isfinite(o.w));
            *(float4 *)(dst + t * 16 + g * 4) = o;
        }
        if (g == 0) {
            if (a.splits > 1)
                *(float2 *)(a.part_ml + at * 2) = make_float2(base, l * 0x1p-14f);
            else if (a.factors)
                a.factors[tile_at(span, s, r0, qh, wide) + i] =
                    kv4_factor(base, l * 0x1p-14f, fbits(qs), a.tops[row * wide + qh]);
        }
        bad |= !(biggest < INFINITY);
    }
    flag_nonfinite(status, bad);
}

// What runs of rows weigh, from their scores once more and the rows' tops and shares: a
// work-group of W waves for 64 keys of a (stream, key head), which stand in each wave's
// registers as fp16; the waves take the tiles of 16 rows that see them in turn. A lane
// adds up its row's weights of 16 keys over the tiles; lanes and waves are added once.
// Bound by the exponentials and the matrix cores: 5 prompts of up to 1777 rows, 16 query
// heads of 64, 42 us, 19 GFLOP with the two terms (4 waves that turned the queries into
// operands themselves: 40 us more).
template <int D, int W>
__global__ __launch_bounds__(64 * W, D == 64 ? 4 : 2) void k_kv4_sums(Kv4 kv, Kv4Rows rows, Kv4Run a,
                                                                      const float *before,
                                                                      float *after, size_t stride,
                                                                      int counted, int *status) {
    constexpr int N = D / kSpan, KS = D / 32;
    __shared__ float parts[W][64];
    const int head = blockIdx.x % kv.heads, c = blockIdx.x / kv.heads, s = blockIdx.z;
    const int wide = kv.heads * a.group;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int i = lane & 15, g = lane >> 4;
    const Kv4Span span = kv4_span(rows, s, a.max_positions, false, status);
    const int end = span.first + span.count;
    if (!span.live || c * 64 >= end) return;
    const int32_t *table = rows.tables + (size_t)s * rows.table_stride;

    int ids[4];
    f16x8 kk[4][KS];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const int b = c * 4 + t;
        ids[t] = b * kBlockPos < end ? uniform_load(table + b) : 0;
        const unsigned id = (unsigned)ids[t] < kv.blocks ? (unsigned)ids[t] : 0u;
        const uint8_t *tl = kv4_tile<D>(kv, id, head);
#pragma unroll
        for (int n = 0; n < N; n++) {
            const u32x2 x = *(const u32x2 *)(tl + n * kPlane + i * 32 + g * 8);
            const uint32_t pair = kv4_scales<D>(kv, id, head)[n * kBlockPos + i];
            // A key that was not finite: no row that sees it counts.
            const f16x2 none = {(_Float16)0.0f, (_Float16)0.0f};
            const f16x2 most = {(_Float16)kMostScale, (_Float16)kMostScale};
            f16x2 s2 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(pair, pair, 0x01000100u));
            s2 = __builtin_elementwise_min(__builtin_elementwise_max(s2, none), most);
#pragma unroll
            for (int k = 0; k < 2; k++) kk[t][n * 2 + k] = word_f16(x[k], s2);
        }
    }

    // Units: a tile of rows, as the attention left it, and a query head of the group.
    const int late = max(0, span.count - counted);  // rows before it do not count
    const int from = max(late, c * 64 - span.first) / 16 * 16;
    const int units = (span.count - from + 15) / 16 * a.group;
    f16x8 nexthi[KS], nextlo[KS];
    float next_top = INFINITY;
    uint32_t next_word = 0;
    // The scores' factors are the scale times powers of two.
    const uint32_t fraction =
        a.scale == 0.0f ? 0 : fbits(fabsf(a.scale) < 1.0f ? a.scale * 0x1p64f : a.scale) & ~(kExponent | kVastRow);
    auto request = [&](int u) {
        const int r0 = from + u / a.group * 16, r = r0 + i, qh = head * a.group + u % a.group;
        const size_t at = tile_at(span, s, r0, qh, wide);
        const uint4 *q = a.queries + at * (D / 4) + lane;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            nexthi[k] = __builtin_bit_cast(f16x8, q[k * 128]);
            nextlo[k] = __builtin_bit_cast(f16x8, q[k * 128 + 64]);
        }
        next_word = a.factors[at + i];
        next_top = a.tops[((size_t)span.row0 + min(r, span.count - 1)) * wide + qh];
        if (r < late || r >= span.count) next_top = INFINITY;
    };
    f32x4 part[4];
#pragma unroll
    for (int t = 0; t < 4; t++) part[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (wave < units) request(wave);
    for (int u = wave; u < units; u += W) {
        const int p0 = span.first + from + u / a.group * 16;
        // Rows that did not come out finite weigh nothing.
        const bool fine = fabsf(next_top) < INFINITY;
        const uint32_t word = next_word;
        const float base = fine ? -next_top : -INFINITY;
        float qs = bitsf((word & kExponent) | fraction);
        float share = bitsf((word & 0x007FFFFFu) | 0x3F000000u);
        f16x8 qhi[KS], qlo[KS];
#pragma unroll
        for (int k = 0; k < KS; k++) qhi[k] = nexthi[k], qlo[k] = nextlo[k];
        if (__any(!fine)) {
            const i32x4 none = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KS; k++)
                if (!fine) qhi[k] = qlo[k] = __builtin_bit_cast(f16x8, none);
            if (!fine) qs = 0.0f;
        }
        if (u + W < units) request(u + W);
        f32x4 w[4];
        auto multiply = [&] {
#pragma unroll
            for (int t = 0; t < 4; t++) w[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; k++) {
#pragma unroll
                for (int t = 0; t < 4; t++)
                    w[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[t][k], qhi[k], w[t], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < 4; t++)
                    w[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[t][k], qlo[k], w[t], 0, 0, 0);
            }
        };
        multiply();
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) w[t][r] = __builtin_amdgcn_exp2f(fmaf(w[t][r], qs, base));
        const bool vast = (int)word < 0, any = __any(vast);
        if (any || c * 64 + 63 > p0) {
            if (any) {  // once more, rounded as the attention did
                multiply();
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        w[t][r] = __builtin_amdgcn_exp2f(vast ? w[t][r] * qs + base : fmaf(w[t][r], qs, base));
                if (vast)
                    share = ldexpf(bitsf((word << 7 & 0x007FFFFFu) | 0x3F000000u),
                                   64 - (int)(word >> 16 & 127));
            }
            const int last = p0 + i - c * 64 - g * 4;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (t * 16 + r > last) w[t][r] = 0.0f;
        }
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) part[t][r] = fmaf(w[t][r], share, part[t][r]);
    }
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float x16 = row16_sum(part[t][r]);
            if (i == 0) parts[wave][t * 16 + g * 4 + r] = x16;
        }
    __syncthreads();
    const int p = c * 64 + (int)threadIdx.x;
    if (threadIdx.x >= 64 || p >= end) return;
    const size_t at = ((size_t)s * kv.heads + head) * stride + p;
    float sum = before && p < span.first ? before[at] : 0.0f;
    const int t = threadIdx.x >> 4, id = t < 2 ? (t ? ids[1] : ids[0]) : (t == 2 ? ids[2] : ids[3]);
    if ((unsigned)id < kv.blocks) {
        float part = 0.0f;
#pragma unroll
        for (int z = 0; z < W; z++) part += parts[z][threadIdx.x];
        sum += part;
    }
    after[at] = sum;
}

// ------------------------------------------------------------------ eviction

// Orders like the number; NaN counts as 0, and -0 as 0.
__device__ inline uint32_t order_of(float x) {
    const uint32_t u = fbits(x == x ? x + 0.0f : 0.0f);
    return u ^ ((int)u < 0 ? 0xFFFFFFFFu : 0x80000000u);
}

constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64, kBins = 2048;

struct Kv4Evict {
    const int32_t *tables, *to_tables;
    int table_stride;
    const int32_t *lengths;
    int keep, first, newest;
    const float *sums;
    float *to_sums;
    size_t sums_stride;
    int32_t *kept;
};

struct Kv4SelectShared {
    uint32_t bins[kBins];
    uint32_t share[2][kEvictWaves];
    uint32_t bin, above, count;
    int bad;
};

// Lane i gets lane i - E's within 16 lanes, the first ones 0; then sums over the lanes up
// to this one, of 16 and of all.
template <int E>
__device__ inline uint32_t row_before(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x110 + E, 0xf, 0xf, false);
}
__device__ inline uint32_t row_scan(uint32_t v) {
    v += row_before<1>(v);
    v += row_before<2>(v);
    v += row_before<4>(v);
    return v + row_before<8>(v);
}
__device__ inline uint32_t wave_scan(uint32_t v) {
    v = row_scan(v);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
}

// The sum over the waves before this one, and (total) over all, of a number of each wave.
// One barrier: `share` is another's until the one after.
__device__ inline uint32_t waves_before(uint32_t *share, uint32_t mine, uint32_t &total) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (lane == 0) share[wave] = mine;
    __syncthreads();
    const uint32_t run = row_scan(share[lane & 15]);
    total = (uint32_t)__builtin_amdgcn_readlane((int)run, kEvictWaves - 1);
    return wave ? (uint32_t)__builtin_amdgcn_readlane((int)run, (wave - 1) & 15) : 0;
}

// What stays: a work-group for each (head, layer, stream). The least order that is kept is
// found digit by digit (11, 11 and 10 bits) from counts in LDS, as far as it takes; then
// the indexes and their sums are dealt out in order. Bound by its chain of barriers and
// what lies between two: 1 stream of 2011 rows 6.0 us, 64 of 600 to 2048 8.9 (8.5 and
// 15.7 with all three digits and sums over the lanes through LDS).
__global__ __launch_bounds__(kEvictThreads) void k_kv4_select(int heads, unsigned blocks,
                                                              Kv4Evict a, int *status) {
    constexpr int H = 8;  // sums that a thread holds
    __shared__ Kv4SelectShared sh;
    const int head = blockIdx.x, layer = blockIdx.y, s = blockIdx.z, streams = gridDim.z;
    const int lane = threadIdx.x & 63;
    const size_t unit = ((size_t)layer * streams + s) * heads + head;
    const float *sums = a.sums + unit * a.sums_stride;
    float *to_sums = a.to_sums + unit * a.sums_stride;
    int32_t *kept = a.kept + unit * a.keep;
    const int32_t *table = a.tables + (size_t)s * a.table_stride;
    const int32_t *to_table = a.to_tables + (size_t)s * a.table_stride;
    const int n = uniform_load(a.lengths + s), count = min(n, a.keep);
    const bool past = n > kMostRows || (n > 0 && ((size_t)n > a.sums_stride ||
                                                  (n - 1) / kBlockPos >= a.table_stride));
    if (threadIdx.x == 0) sh.bad = past;
    for (int b = threadIdx.x; b < kBins; b += kEvictThreads) sh.bins[b] = 0;
    __syncthreads();
    // The sums of rows threadIdx.x + 1024 k.
    float held[H];
#pragma unroll
    for (int k = 0; k < H; k++) {
        const int i = threadIdx.x + k * kEvictThreads;
        held[k] = !past && i < n ? sums[i] : 0.0f;
    }
    if (!past && n > 0) {
        bool bad = false;
        for (int b = threadIdx.x; b * kBlockPos < n; b += kEvictThreads) {
            bad |= (unsigned)table[b] >= blocks;
            if (b * kBlockPos < count) bad |= (unsigned)to_table[b] >= blocks;
        }
        if (bad) sh.bad = 1;
    }
    __syncthreads();
    if (sh.bad || n <= 0) {
        for (int j = threadIdx.x; j < a.keep; j += kEvictThreads) kept[j] = -1;
        if (sh.bad && threadIdx.x == 0) atomicOr(status, 2);
        return;
    }

    const int lo = n > a.keep ? a.first : n, hi = n > a.keep ? n - a.newest : n;
    uint32_t need = n > a.keep ? a.keep - a.first - a.newest : 0, least = 0;
    const bool choose = need != 0;
    auto count_digit = [&](int i, float x, int shift, int width) {
        const uint32_t u = order_of(x);
        if (i >= lo && i < hi && (shift == 32 || (u >> shift) == (least >> shift)))
            atomicAdd(&sh.bins[u >> (shift - width) & ((1u << width) - 1)], 1u);
    };
    // Orders from `from` on are kept, and of those equal to `least` the first `need`.
    uint32_t from = 0;
    if (choose) {
        int shift = 32;
        for (int digit = 0; digit < 3; digit++) {
            const int width = digit < 2 ? 11 : 10;
#pragma unroll
            for (int k = 0; k < H; k++)
                if (k * kEvictThreads < n) count_digit(threadIdx.x + k * kEvictThreads, held[k], shift, width);
            for (int i = threadIdx.x + H * kEvictThreads; i < hi; i += kEvictThreads)
                count_digit(i, sums[i], shift, width);
            __syncthreads();
            // Two bins to a thread, from the top; cleared for the next digit.
            const int b = kBins - 1 - 2 * (int)threadIdx.x;
            const uint32_t x = sh.bins[b], y = sh.bins[b - 1];
            sh.bins[b] = sh.bins[b - 1] = 0;
            const uint32_t run = wave_scan(x + y);
            uint32_t total;
            const uint32_t before =
                waves_before(sh.share[digit & 1], __builtin_amdgcn_readlane((int)run, 63), total) +
                run - x - y;
            if (before < need && before + x >= need) {
                sh.bin = b;
                sh.above = before;
                sh.count = x;
            } else if (before + x < need && before + x + y >= need) {
                sh.bin = b - 1;
                sh.above = before + x;
                sh.count = y;
            }
            __syncthreads();
            shift -= width;
            least |= sh.bin << shift;
            need -= sh.above;
            from = least + 1;  // not past 2^32: orders end at infinity's
            if (need == sh.count) {  // the whole bin
                from = least;
                need = 0;
                break;
            }
        }
    }
    // The indexes and their sums, in order. A row comes after those before it that are
    // larger (or not to be chosen among) and as many of the equal ones as are kept.
    uint32_t larger = 0, equal = 0;
    auto place = [&](int round, float x) {
        const int i = threadIdx.x + round * kEvictThreads;
        const uint32_t u = order_of(x);
        const bool middle = i >= lo && i < hi;
        const bool more = i < n && (!middle || (choose && u >= from)), same = need && middle && u == least;
        const uint64_t up = __ballot(more), eq = __ballot(same), below = (1ull << lane) - 1;
        uint32_t total;
        const uint32_t before = waves_before(sh.share[round & 1],
                                             (uint32_t)(__popcll(up) | __popcll(eq) << 16), total);
        const uint32_t rank = equal + (before >> 16) + __popcll(eq & below);
        if (more || (same && rank < need)) {
            const uint32_t to = larger + (before & 0xFFFFu) + __popcll(up & below) + min(rank, need);
            kept[to] = i;
            to_sums[to] = x == x ? x : 0.0f;
        }
        larger += total & 0xFFFFu;
        equal += total >> 16;
    };
#pragma unroll
    for (int k = 0; k < H; k++)
        if (k * kEvictThreads < n) place(k, held[k]);
    for (int k = H; k * kEvictThreads < n; k++) {
        const int i = threadIdx.x + k * kEvictThreads;
        place(k, i < n ? sums[i] : 0.0f);
    }
    for (int j = count + threadIdx.x; j < a.keep; j += kEvictThreads) kept[j] = -1;
}

// Waits for this wave's loads.
__device__ inline void loads_done() { __builtin_amdgcn_s_waitcnt(0xF70); }

// The kept rows to their places: a work-group for each (head; keys with the scales, or
// values, of 64 dims; layer, stream), which moves 4 blocks of keys or one of values to a
// wave between two barriers. A block's rows come from its own place or later ones, and
// all that are read before a barrier are written after it, so that nothing is read that
// was written. Past the last row: the last one again. A row's 32 bytes of keys are four
// lanes' words. Values lie by dim: a lane takes its dim's 16 numbers of each source block,
// once where rows side by side are of one, and picks those that stay. Bound by memory
// where there is much to move: 64 streams of 600 to 2048 rows shrunk to 1024, 86 MB by
// the counters, 25 us (41 with a word loaded for each row, 13 cycles of the L1 cache each;
// 4 blocks at a time of each source block in a loop: 36). With 8 waves evictions of 64
// streams take as long, of 2 of up to 6156 rows 52 us with the rows read back, not 43.
template <int D>
__global__ __launch_bounds__(kEvictThreads, 8) void k_kv4_move(Kv4 kv, size_t layer_values,
                                                               size_t layer_scales, Kv4Evict a) {
    constexpr int N = D / kSpan;
    const int head = blockIdx.x % kv.heads, part = blockIdx.x / kv.heads, m = part % N;
    const int layer = blockIdx.y, s = blockIdx.z, streams = gridDim.z;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    kv.values += layer * layer_values;
    kv.scales += layer * layer_scales;
    const int32_t *kept = a.kept + (((size_t)layer * streams + s) * kv.heads + head) * a.keep;
    const int32_t *table = a.tables + (size_t)s * a.table_stride;
    const int32_t *to_table = a.to_tables + (size_t)s * a.table_stride;
    const int n = uniform_load(a.lengths + s), count = min(n, a.keep);
    // Left out, or whole and in place.
    if (count <= 0 || uniform_load(kept) < 0 || (n <= a.keep && a.to_tables == a.tables)) return;
    const int j = lane >> 2;

    // Row j of a wave's e-th block of the round from block b0 on.
    struct Row {
        int at, src;
        unsigned id, to;
    };
    auto find = [&](int b0, int e) {
        Row x;
        x.at = min((b0 + e * kEvictWaves + wave) * kBlockPos + j, count - 1);
        x.src = kept[x.at];
        x.to = (unsigned)to_table[x.at / kBlockPos];
        x.id = 0;
        return x;
    };
    // Whether there is a block to write: not past the last, and not where it belongs.
    auto moves = [&](const Row &x, int b0, int e) {
        return (b0 + e * kEvictWaves + wave) * kBlockPos < count &&
               !__all(x.id == x.to && x.src == x.at);
    };

    if (part < N) {
        constexpr int K = 4;
        Row x[K];
#pragma unroll
        for (int e = 0; e < K; e++) x[e] = find(0, e);
#pragma unroll
        for (int e = 0; e < K; e++) x[e].id = (unsigned)table[x[e].src / kBlockPos];
        for (int b0 = 0; b0 * kBlockPos < count; b0 += kEvictWaves * K) {
            uint64_t key[K];
            uint32_t pair[K];
#pragma unroll
            for (int e = 0; e < K; e++) {
                const int row = x[e].src % kBlockPos;
                key[e] = *((const uint64_t *)(kv4_tile<D>(kv, x[e].id, head) + m * kPlane +
                                              row * (kSpan / 2)) + (lane & 3));
                pair[e] = kv4_scales<D>(kv, x[e].id, head)[m * kBlockPos + row];
            }
            Row next[K];
#pragma unroll
            for (int e = 0; e < K; e++) next[e] = find(b0 + kEvictWaves * K, e);
#pragma unroll
            for (int e = 0; e < K; e++) next[e].id = (unsigned)table[next[e].src / kBlockPos];
            loads_done();
            __syncthreads();
#pragma unroll
            for (int e = 0; e < K; e++) {
                if (moves(x[e], b0, e) && (b0 + e * kEvictWaves + wave) * kBlockPos + j < count) {
                    *((uint64_t *)(kv4_tile<D>(kv, x[e].to, head) + m * kPlane + j * (kSpan / 2)) +
                      (lane & 3)) = key[e];
                    if ((lane & 3) == 0) kv4_scales<D>(kv, x[e].to, head)[m * kBlockPos + j] = pair[e];
                }
                x[e] = next[e];
            }
        }
        return;
    }
    Row x = find(0, 0);
    x.id = (unsigned)table[x.src / kBlockPos];
    for (int b0 = 0; b0 * kBlockPos < count; b0 += kEvictWaves) {
        uint64_t w[kBlockPos];
        const int last = __shfl_up(x.src, 4);
        // Bit 4 r: row r is the first of its source block.
        uint64_t starts = __ballot(lane < 4 || x.src / kBlockPos != last / kBlockPos);
        const uint64_t tile = (uint64_t)(kv4_tile<D>(kv, x.id, head) + (N + m) * kPlane);
#pragma unroll
        for (int r = 0; r < kBlockPos; r++)
            if (starts >> (4 * r) & 1) {
                const uint64_t low = (uint32_t)__builtin_amdgcn_readlane((int)tile, r * 4);
                const uint64_t high = (uint32_t)__builtin_amdgcn_readlane((int)(tile >> 32), r * 4);
                w[r] = ((const __attribute__((address_space(1))) uint64_t *)(high << 32 | low))[lane];
            }
        Row next = find(b0 + kEvictWaves, 0);
        // Not known to be the loads' conditions: they would wait for one another.
        asm("" : "+s"(starts));
        // Where a row's number stands among its dim's 64 bits.
        const int bit = (x.src & 3) * 8 + (x.src & 4) + (x.src & 8) * 4;
        uint64_t here = w[0];
        uint32_t dim[2] = {0, 0};
#pragma unroll
        for (int r = 0; r < kBlockPos; r++) {
            if (starts >> (4 * r) & 1) here = w[r];
            const uint32_t number = (uint32_t)(here >> __builtin_amdgcn_readlane(bit, r * 4)) & 15u;
            dim[r >> 3] |= number << ((r & 3) * 8 + (r & 4));
        }
        next.id = (unsigned)table[next.src / kBlockPos];
        loads_done();
        __syncthreads();
        if (moves(x, b0, 0))
            *((uint2 *)(kv4_tile<D>(kv, (unsigned)__builtin_amdgcn_readfirstlane(x.to), head) +
                        (N + m) * kPlane) + lane) = make_uint2(dim[0], dim[1]);
        x = next;
    }
}

}  // namespace pgpu

using namespace pgpu;

// ------------------------------------------------------------- entry points

namespace {

bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

bool cache_ok(const pgpu_kv4 *kv) {
    return kv && kv->values && kv->scales && aligned(kv->values, 16) && aligned(kv->scales, 16) &&
           kv->layers > 0 && kv->heads > 0 && kv->heads <= 256 &&
           (kv->head_dim == 64 || kv->head_dim == 128) && kv->blocks > 0 &&
           kv->blocks <= INT32_MAX;
}

bool rows_ok(const pgpu_kv4_rows *r) {
    return r && r->tables && r->table_stride > 0 && r->first && r->streams > 0 &&
           r->streams <= 65535 && r->rows >= 0 && r->max_rows >= 0 && r->max_rows <= 65535 &&
           r->max_rows <= r->rows &&
           (r->offsets ? (r->max_rows > 0 || r->rows == 0)
                       : (r->rows == r->streams && r->max_rows == 1));
}

// Bytes of a layer, and its scale pairs.
size_t layer_values(const pgpu_kv4 *kv) {
    return kv->blocks * kv->heads * kv->head_dim * kBlockPos;
}
size_t layer_scales(const pgpu_kv4 *kv) {
    return kv->blocks * kv->heads * (kv->head_dim / kSpan) * kBlockPos;
}

Kv4 layer_of(const pgpu_kv4 *kv, int layer) {
    return {kv->values + layer * layer_values(kv), (uint32_t *)kv->scales + layer * layer_scales(kv),
            kv->heads, (unsigned)kv->blocks};
}

Kv4Rows rows_of(const pgpu_kv4_rows *r) {
    return {r->tables, r->table_stride, r->first, r->offsets, r->rows, r->max_rows};
}

// Blocks that max_rows consecutive rows can lie in.
int blocks_of(int max_rows) { return (max_rows + 2 * kBlockPos - 2) / kBlockPos; }

}  // namespace

extern "C" int pgpu_kv4_write(void *stream, const pgpu_kv4 *kv, int layer,
                              const pgpu_kv4_rows *rows, const float *k, const float *v,
                              size_t row_stride, int *status) {
    if (!cache_ok(kv) || !rows_ok(rows) || layer < 0 || layer >= kv->layers || !k || !v ||
        !status || !aligned(k, 16) || !aligned(v, 16) || row_stride % 4 != 0 ||
        row_stride < (size_t)kv->heads * kv->head_dim)
        return bad_arguments("pgpu_kv4_write");
    if (rows->rows == 0) return 1;
    const dim3 grid((kv->heads + 3) / 4, blocks_of(rows->max_rows), rows->streams);
    if (kv->head_dim == 64)
        hipLaunchKernelGGL(k_kv4_write<64>, grid, dim3(256), 0, (hipStream_t)stream,
                           layer_of(kv, layer), rows_of(rows), k, v, row_stride, status);
    else
        hipLaunchKernelGGL(k_kv4_write<128>, grid, dim3(256), 0, (hipStream_t)stream,
                           layer_of(kv, layer), rows_of(rows), k, v, row_stride, status);
    return launch_ok("pgpu_kv4_write");
}

extern "C" int pgpu_kv4_read(void *stream, const pgpu_kv4 *kv, int layer,
                             const pgpu_kv4_rows *rows, const int32_t *lengths, float *k,
                             float *v, size_t row_stride, int *status) {
    if (!cache_ok(kv) || !rows_ok(rows) || layer < 0 || layer >= kv->layers || !lengths || !k ||
        !v || !status || !aligned(k, 16) || !aligned(v, 16) || row_stride % 4 != 0 ||
        row_stride < (size_t)kv->heads * kv->head_dim)
        return bad_arguments("pgpu_kv4_read");
    if (rows->rows == 0) return 1;
    const dim3 grid((kv->heads + 3) / 4, blocks_of(rows->max_rows), rows->streams);
    if (kv->head_dim == 64)
        hipLaunchKernelGGL(k_kv4_read<64>, grid, dim3(256), 0, (hipStream_t)stream,
                           layer_of(kv, layer), rows_of(rows), lengths, k, v, row_stride, status);
    else
        hipLaunchKernelGGL(k_kv4_read<128>, grid, dim3(256), 0, (hipStream_t)stream,
                           layer_of(kv, layer), rows_of(rows), lengths, k, v, row_stride, status);
    return launch_ok("pgpu_kv4_read");
}

namespace {

// The cache rows that a call can count. A run's sums: the grid's 2^32 threads.
bool positions_ok(const pgpu_kv4 *kv, const pgpu_kv4_rows *rows, int max_positions, bool sums) {
    if (!rows->offsets) return max_positions > 0 && max_positions <= kMostOne;
    return max_positions > 0 && max_positions <= kMostRows &&
           !(sums && kv->heads * (size_t)((max_positions + 63) / 64) >= (size_t)1 << 22);
}

// How an attention call deals its work: splits of `keys` keys.
struct Deal {
    int splits, keys, tiles, waves, steps;  // tiles: work-groups for a stream and head
};

Deal deal_rows(const pgpu_kv4 *kv, const pgpu_kv4_rows *r, int group, int max_positions) {
    // Work-groups without splits. Where they are few, and the keys enough to pay for the
    // join, each row's keys are dealt out in chunks of 64: of 64 work-groups at most to
    // 1024 of them, of more to 4 splits (or 512 work-groups).
    // us a pass (9.5 at least with two launches), 8 heads, whole / dealt. Few rows, heads of 64
    // and of 128: 60 of 1 stream behind 180 keys 9.4 / 9.6, 12.7 / 11.1; behind 320 11.9 / 9.6, 16.5 / 11.4; behind 1000 25.5 / 9.5,
    // 36.3 / 11.9; behind 8000 159 / 13.4, 230 / 19.3; 8 streams behind 4000 83.6 / 25.2, 120 /
    // 39.6; 1 of 300 rows 10.4 / 11.0, 14.3 / 14.7. More: 16 streams of 64 behind 450 15.4 /
    // 18.1, 21.8 / 22.8, behind 700 19.0 / 18.0, 27.2 / 23.1, behind 2000 44.0 / 25.9, 63.7 /
    // 37.7; 1 of 600 rows 16.6 / 14.2, 23.3 / 20.4; of 2000 41.1 / 26.1, 60.2 / 43.5.
    // Splits 1 / 2 / 4 / 8 / 16: 16 streams of 64 behind 2000 44.0 / 30.8 / 25.5 / 26.2 / 34.6;
    // 1 of 2000 41.1 / 32.3 / 25.7 / 31.1 / 47.1. More than 512 work-groups: 1 of 8187 rows,
    // 1 / 2 splits 182 / 173, whose parts take 69 MB: not taken; 4 of 2000 56.9 / 67.1.
    Deal d = {};
    d.tiles = ((r->max_rows + 15) / 16 * group + 3) / 4;
    const size_t groups = (size_t)d.tiles * kv->heads * r->streams;
    const int chunks = (max_positions - 1) / 64 + 1;
    d.splits = 1;
    if (groups < 512 && chunks > (groups > 64 ? 9 : groups > 32 || kv->head_dim == 64 ? 5 : 3)) {
        d.splits = std::min(groups > 32 ? chunks / 2 : chunks, (int)(1024 / groups));
        if (groups > 64) d.splits = std::min(d.splits, std::max(4, (int)(512 / groups)));
        if (d.splits > 32) d.splits = 32;
    }
    return d;
}

Deal deal_of(const pgpu_kv4 *kv, int streams, int group, int max_positions) {
    Deal d;
    // A stream's keys whole in one work-group of W waves (no parts to be joined), except
    // where few work-groups have many keys each, or contexts are long enough to differ
    // much: those are dealt to work-groups of 4 waves, in steps of W * 64 keys, more to
    // each the more of them there are.
    // us, 8 heads (contexts of one stream as said, of several up to that), whole / dealt
    // with the steps taken here. Heads of 64: 1 stream of 2048 keys 7.5 / 10.1, of 8187
    // 16.8 / 10.1; 16 of 4096 10.6 / 11.1, of 8187 17.4 / 13.0; 32 of 4096 11.2 / 14.6, of
    // 8187 18.9 / 19.2; 64 of 4096 18.8 / 20.5, of 6000 22.6 / 23.7, of 8187 34.0 / 28.8;
    // 256 of 8187 101.2 / 98.5; 4 queries each: 4 of 4096 13.8 / 10.2, 16 of 2900 11.4 /
    // 11.5, of 8187 23.4 / 15.5, 64 of 8187 34.9 / 33.2. Heads of 128: 1 of 2048 9.7 / 10.2,
    // 16 of 8187 29.8 / 19.4, 48 of 4096 29.7 / 24.5, 128 54.2 / 51.3; 4 queries each: 1 of
    // 2048 12.5 / 10.0, 16 of 2900 16.4 / 15.5, 48 of 4096 34.0 / 28.9, 64 of 2048 21.5 / 31.
    // Steps of a dealt work-group, 1 / 2 / 3 / 4 / 5: heads of 64, 16 of 8187 15.4 / 13.0 /
    // 14.4 / 14.7 / 14.0, 64 38.7 / 29.6 / 29.0 / 28.8 / 28.9; heads of 128 with 4 queries,
    // 4 of 4096 11.2 / 10.9 / 12.3 / 13.7 / 14.9, 16 of 2900 17.0 / 16.2 / 15.5 / 17.3 / 19.0,
    // 48 of 4096 38.2 / 31.0 / 30.6 / 30.7 / 28.9.
    // W = 4 / 8: heads of 64, 64 streams of 2048 11.1 / 11.4, of 6000 23.9 / 22.6, 128 of
    // 2048 18.3 / 19.3, with 4 queries 64 of 2048 14.1 / 13.5; heads of 128, 64 of 600 8.6 /
    // 9.9, with 4 queries 10.9 / 13.7. (W = 16: 1 of 2048 7.5, 64 of 2048 13.9.)
    d.tiles = group == 1 ? 1 : (group + 3) / 4;
    const size_t groups = (size_t)kv->heads * d.tiles * streams;
    const int units = (max_positions - 1) / 64 + 1;
    const bool wide = kv->head_dim != 64, four = group > 1, both = wide && four;
    d.waves = groups >= 512 && units <= 64 && (wide || !four) ? 4 : 8;
    d.steps = (units + d.waves - 1) / d.waves;
    if (units > (groups >= 192 ? (wide ? 48 : 96) : both ? 24 : wide || four ? 48 : 64)) {
        d.waves = 4;
        d.steps = groups < 64 ? 1 : groups < 192 ? (both ? 3 : 2) : both ? 5 : 4;
    }
    d.keys = 64 * d.waves * d.steps;
    d.splits = (max_positions - 1) / d.keys + 1;
    return d;
}

// The workspace of one row a stream: parts of `parts` (row, query head, split), then the
// rows' tops and shares, and their scores.
size_t parts_bytes(const pgpu_kv4 *kv, size_t parts) {
    return parts * (kv->head_dim + 2) * sizeof(float);
}

// What a run's sums need: the queries as operands, their words and the rows' tops (and room
// to align what follows).
size_t run_sums_bytes(const pgpu_kv4 *kv, const pgpu_kv4_rows *r, int group) {
    const size_t wide = (size_t)kv->heads * group;
    return ((r->rows + (size_t)16 * r->streams) * wide * (kv->head_dim + 1) + r->rows * wide + 4) *
           sizeof(float);
}

template <int D>
int join(hipStream_t st, const Kv4 &c, const Kv4Rows &r, int streams, const Deal &d,
         const float *part_acc, const float *part_ml, int group, int max_positions, float *out,
         size_t out_stride, float *tops, float *shares, uint32_t *factors, int *status) {
    // Many splits of few rows: a wave for each, spread over the CUs; else few splits of
    // many rows. us with the attention, 8 heads of 64: 60 rows behind 8000 keys 13.2 / 17.6, 8
    // streams of them behind 4000 24.0 / 25.7, a row behind 8186 9.4 / 9.9; 2000 rows (4
    // splits) 30.3 / 25.3; heads of 128, 16 streams of 64 behind 2000 39.0 / 36.9.
    const size_t items = (size_t)r.max_rows * c.heads * group;
    if (d.splits >= 8 && items * streams <= 4096)
        hipLaunchKernelGGL((k_kv4_join<D, 256 / D>), dim3((unsigned)items, 1, streams), dim3(64), 0,
                           st, c, r, part_acc, part_ml, group, max_positions, d.splits, d.keys, out,
                           out_stride, tops, shares, factors, status);
    else
        hipLaunchKernelGGL((k_kv4_join<D, 1>),
                           dim3((unsigned)((items * (D / 4) + 255) / 256), 1, streams), dim3(256), 0,
                           st, c, r, part_acc, part_ml, group, max_positions, d.splits, d.keys, out,
                           out_stride, tops, shares, factors, status);
    return launch_ok("pgpu_kv4_attention");
}

template <int D>
int attend_one(hipStream_t st, const Kv4 &c, const Kv4Rows &r, int streams, const Deal &d,
               const Kv4Decode &a, const pgpu_kv4_sums *sums, int *status) {
    Kv4Decode one = a;
    one.steps = d.steps;
    if (d.splits > 1) one.out = nullptr;
    // The weights are added up where a work-group has all of a key's.
    if (sums && d.splits == 1 && d.tiles == 1) one.after = sums->after;
    const dim3 grid(c.heads * d.tiles, d.splits, streams);
#define KV4_DECODE(W, Q)                                                                        \
    do {                                                                                        \
        if (sums)                                                                               \
            hipLaunchKernelGGL((k_kv4_decode<D, W, Q, true>), grid, dim3(64 * W), 0, st, c, r,  \
                               one, status);                                                    \
        else                                                                                    \
            hipLaunchKernelGGL((k_kv4_decode<D, W, Q, false>), grid, dim3(64 * W), 0, st, c, r, \
                               one, status);                                                    \
    } while (0)
    if (a.group == 1 && d.waves == 4)
        KV4_DECODE(4, 1);
    else if (a.group == 1)
        KV4_DECODE(8, 1);
    else if (d.waves == 4)
        KV4_DECODE(4, 4);
    else
        KV4_DECODE(8, 4);
#undef KV4_DECODE
    if (!launch_ok("pgpu_kv4_attention")) return 0;
    if (d.splits > 1 && !join<D>(st, c, r, streams, d, a.part_acc, a.part_ml, a.group,
                                 a.max_positions, a.out, a.out_stride, a.tops, a.shares, nullptr,
                                 status))
        return 0;
    if (!sums || one.after) return 1;
    one.after = sums->after;
    hipLaunchKernelGGL(k_kv4_sums_one, dim3((a.max_positions + 255) / 256, c.heads, streams),
                       dim3(256), 0, st, c, r, one, status);
    return launch_ok("pgpu_kv4_attention");
}

template <int D>
int attend_rows(hipStream_t st, const Kv4 &c, const Kv4Rows &r, int streams, const Deal &d,
                const Kv4Run &a, const pgpu_kv4_sums *sums, int *status) {
    hipLaunchKernelGGL(k_kv4_run<D>, dim3(c.heads * d.splits, d.tiles, streams), dim3(256), 0, st, c,
                       r, a, status);
    if (!launch_ok("pgpu_kv4_attention")) return 0;
    if (d.splits > 1 && !join<D>(st, c, r, streams, d, a.part_acc, a.part_ml, a.group,
                                 a.max_positions, a.out, a.out_stride, a.tops, nullptr, a.factors,
                                 status))
        return 0;
    if (!sums) return 1;
    constexpr int W = D == 64 ? 16 : 8;
    hipLaunchKernelGGL((k_kv4_sums<D, W>), dim3(c.heads * (unsigned)((a.max_positions + 63) / 64), 1,
                                                streams),
                       dim3(64 * W), 0, st, c, r, a, sums->before, sums->after, sums->stride,
                       sums->rows, status);
    return launch_ok("pgpu_kv4_attention");
}

}  // namespace

extern "C" size_t pgpu_kv4_attention_bytes(const pgpu_kv4 *kv, const pgpu_kv4_rows *rows,
                                           int group, int max_positions, int with_sums) {
    if (!cache_ok(kv) || !rows_ok(rows) || group < 1 || group > 16 ||
        !positions_ok(kv, rows, max_positions, with_sums != 0))
        return 0;
    const size_t wide = (size_t)kv->heads * group;
    if (rows->rows == 0) return 0;
    size_t parts = 0;
    if (rows->offsets) {
        // Fewer rows or positions may be dealt to more work-groups. Splits times
        // work-groups are at most 1024, a work-group has 64 rows.
        const int chunks = (max_positions - 1) / 64 + 1;
        const int most = std::min({32, chunks <= 3 ? 1 : chunks,
                                   1024 / (kv->heads * ((group + 3) / 4))});
        if (most > 1)
            parts = std::min((size_t)1024 * 64, (size_t)rows->streams * rows->max_rows * wide * most);
        return parts_bytes(kv, parts) + (with_sums ? run_sums_bytes(kv, rows, group) : 0);
    }
    // Fewer streams may be dealt to more work-groups: the streams before the numbers of
    // work-groups where the keys to each change count too. More positions never give
    // fewer parts.
    const int groups = kv->heads * (group == 1 ? 1 : (group + 3) / 4);
    for (int n : {rows->streams, 63 / groups, 191 / groups}) {
        if (n < 1 || n > rows->streams) continue;
        const Deal d = deal_of(kv, n, group, max_positions);
        if (d.splits > 1) parts = std::max(parts, n * wide * d.splits);
    }
    return parts_bytes(kv, parts) +
           (with_sums ? rows->streams * wide * (2 + (size_t)max_positions) * sizeof(float) : 0);
}

extern "C" int pgpu_kv4_attention(void *stream, const pgpu_kv4 *kv, int layer,
                                  const pgpu_kv4_rows *rows, const float *q, size_t q_stride,
                                  int group, float scale, int max_positions, float *out,
                                  size_t out_stride, const pgpu_kv4_sums *sums, void *work,
                                  size_t work_bytes, int *status) {
    constexpr float kLog2e = 1.44269504f;
    const size_t width = kv ? (size_t)kv->heads * kv->head_dim * group : 0;
    if (!cache_ok(kv) || !rows_ok(rows) || layer < 0 || layer >= kv->layers || !q || !out ||
        !status || !aligned(q, 16) || !aligned(out, 16) || q_stride % 4 != 0 ||
        out_stride % 4 != 0 || group < 1 || group > 16 || q_stride < width ||
        out_stride < width || !positions_ok(kv, rows, max_positions, sums != nullptr) ||
        !__builtin_isfinite(scale * kLog2e) ||
        (sums && (!sums->after || sums->stride < (size_t)max_positions || sums->rows < 1)))
        return bad_arguments("pgpu_kv4_attention");
    if (rows->rows == 0) return 1;
    const Kv4 c = layer_of(kv, layer);
    const Kv4Rows r = rows_of(rows);
    const hipStream_t st = (hipStream_t)stream;
    const size_t wide = (size_t)kv->heads * group;
    float *floats = (float *)work;
    if (!rows->offsets) {
        const Deal d = deal_of(kv, rows->streams, group, max_positions);
        const size_t parts = d.splits > 1 ? rows->streams * wide * d.splits : 0;
        const size_t need = parts_bytes(kv, parts) +
                            (sums ? rows->streams * wide * (2 + (size_t)max_positions) * sizeof(float)
                                  : 0);
        if (need && (!work || !aligned(work, 16) || work_bytes < need))
            return bad_arguments("pgpu_kv4_attention (workspace)");
        Kv4Decode a = {};
        a.q = q;
        a.q_stride = q_stride;
        a.group = group;
        a.scale = scale * kLog2e;
        a.max_positions = max_positions;
        a.splits = d.splits;
        a.part_acc = floats;
        a.part_ml = floats + parts * kv->head_dim;
        a.out = out;
        a.out_stride = out_stride;
        if (sums) {
            a.tops = floats + parts * (kv->head_dim + 2);
            a.shares = a.tops + rows->streams * wide;
            a.scores = a.shares + rows->streams * wide;
            a.before = sums->before;
            a.stride = sums->stride;
        }
        return kv->head_dim == 64 ? attend_one<64>(st, c, r, rows->streams, d, a, sums, status)
                                  : attend_one<128>(st, c, r, rows->streams, d, a, sums, status);
    }
    const Deal d = deal_rows(kv, rows, group, max_positions);
    const size_t parts = d.splits > 1 ? (size_t)rows->streams * rows->max_rows * wide * d.splits : 0;
    const size_t need = parts_bytes(kv, parts) + (sums ? run_sums_bytes(kv, rows, group) : 0);
    if (need && (!work || !aligned(work, 16) || work_bytes < need))
        return bad_arguments("pgpu_kv4_attention (workspace)");
    Kv4Run a = {};
    a.q = q;
    a.q_stride = q_stride;
    a.group = group;
    a.scale = scale * kLog2e;
    a.max_positions = max_positions;
    a.splits = d.splits;
    a.out = out;
    a.out_stride = out_stride;
    if (sums) {
        const size_t slots = (rows->rows + (size_t)16 * rows->streams) * wide;
        a.queries = (uint4 *)floats;
        a.factors = (uint32_t *)(floats + slots * kv->head_dim);
        a.tops = floats + slots * (kv->head_dim + 1);
        a.counted = sums->rows;
        floats = a.tops + rows->rows * wide;
    }
    a.part_acc = floats + (-(uintptr_t)floats / sizeof(float) & 3);
    a.part_ml = a.part_acc + parts * kv->head_dim;
    return kv->head_dim == 64 ? attend_rows<64>(st, c, r, rows->streams, d, a, sums, status)
                              : attend_rows<128>(st, c, r, rows->streams, d, a, sums, status);
}

extern "C" int pgpu_kv4_evict(void *stream, const pgpu_kv4 *kv, int first_layer, int layers,
                              const int32_t *tables, const int32_t *to_tables, int table_stride,
                              const int32_t *lengths, int streams, int keep, int first,
                              int newest, const float *sums, float *to_sums,
                              size_t sums_stride, int32_t *kept, int *status) {
    if (!cache_ok(kv) || first_layer < 0 || layers <= 0 || first_layer > kv->layers - layers ||
        layers > 65535 || !tables || table_stride <= 0 || !lengths || streams <= 0 ||
        streams > 65535 || keep < 1 || keep > kMostRows || first < 0 || newest < 0 || first > keep - newest || !sums ||
        !to_sums || sums_stride == 0 || !kept || !status)
        return bad_arguments("pgpu_kv4_evict");
    const Kv4Evict a = {tables, to_tables ? to_tables : tables, table_stride, lengths, keep, first,
                        newest, sums, to_sums, sums_stride, kept};
    const hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(k_kv4_select, dim3(kv->heads, layers, streams), dim3(kEvictThreads), 0, st,
                       kv->heads, (unsigned)kv->blocks, a, status);
    if (!launch_ok("pgpu_kv4_evict")) return 0;
    const dim3 grid(kv->heads * 2 * (kv->head_dim / kSpan), layers, streams);
    if (kv->head_dim == 64)
        hipLaunchKernelGGL(k_kv4_move<64>, grid, dim3(kEvictThreads), 0, st,
                           layer_of(kv, first_layer), layer_values(kv), layer_scales(kv), a);
    else
        hipLaunchKernelGGL(k_kv4_move<128>, grid, dim3(kEvictThreads), 0, st,
                           layer_of(kv, first_layer), layer_values(kv), layer_scales(kv), a);
    return launch_ok("pgpu_kv4_evict");
}
