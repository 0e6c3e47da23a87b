// kvcache.hip -- a paged key/value cache held in 8 bits, and the operators of
// a decode or prompt step on it: append, read, select, attend, evict.
//
// No counterpart in the reference.  The timing engine prices the reads and
// writes of a paged cache (the paged-KV record streams of workloads.py); these
// operators are the step itself, so that a study knows which blocks a step
// reads, which may leave for the flash tier, and what the tokens become.
//
// Layout.  A block holds t tokens (16, 32, 64 or 128) of every kv head; P is
// the head dimension rounded up to 64.  Per (block, kv head) the codes are
// t/16 tiles of 16 tokens x P dims, and a tile's 1-KiB pieces (16 tokens x 64
// dims) are stored in the order in which a wave's lanes feed them to the
// matrix units, so one 16-byte load per lane fetches a whole piece from one
// contiguous KiB and nothing is transposed in LDS or registers:
//   keys   lane (c, t): token t, dims 16 c .. 16 c + 15 of the piece
//   values lane (c, n): tokens 4 c .. 4 c + 3 of dims n, 16 + n, 32 + n, 48 + n
// with lane = 16 c + t.  Scores are computed as S^T = K Q^T (a lane holds one
// query row's scores of tokens 4 c .. 4 c + 3), which is already the operand
// layout in which O^T = V^T P^T wants the probabilities.
//
// Codes are widened to f16 (exact) and multiplied in f16 with f32 sums: a
// query row is first scaled by a power of two so that its largest element
// lies in [2^14, 2^15), where a bf16 or f16 value keeps every bit down to
// 2^-28 of the row's largest.  A block's value scale joins the exponent: with
//   t = score + log2(value_scale),  w = 2^(t - m)
// the row's output is sum(w code) / sum(w / value_scale), so one set of
// accumulators serves blocks of different scales.  Sums, maxima and
// denominators are f32; w is rounded to f16 (11 bits) for the matrix units,
// finer than the output types' own rounding of bf16 and equal to f16's.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "../../include/hbfsim_amd.h"

#include <cstddef>
#include <cstdint>
#include <type_traits>

namespace {

constexpr int kWave = 64;
constexpr int kPickThreads = 1024;  // of a workgroup that chooses blocks
constexpr float kInv127 = 1.0f / 127.0f;
constexpr float kScaleMin = 0x1p-40f;
constexpr float kScaleMax = 0x1p40f;
constexpr float kQueryScaleMin = 0x1p-100f;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();
constexpr float kLowest = -3.0e38f;            // a row's reference exponent before its first score
constexpr std::int32_t kNowhere = 0x7fffffff - 127;  // a position that no row sees

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef std::int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef std::uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Bf16 {
    std::uint16_t bits;
};
struct F16 {
    std::uint16_t bits;
};

__device__ inline float to_float(Bf16 x)
{
    return __uint_as_float(static_cast<std::uint32_t>(x.bits) << 16);
}
__device__ inline float to_float(F16 x) { return static_cast<float>(__builtin_bit_cast(_Float16, x.bits)); }
__device__ inline float to_float(float x) { return x; }

template <typename T>
__device__ inline T from_float(float x);
template <>
__device__ inline Bf16 from_float<Bf16>(float x)
{
    const std::uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) {
        return Bf16{static_cast<std::uint16_t>((u >> 16) | 0x40u)};
    }
    return Bf16{static_cast<std::uint16_t>((u + 0x7fffu + ((u >> 16) & 1u)) >> 16)};
}
template <>
__device__ inline F16 from_float<F16>(float x)
{
    return F16{__builtin_bit_cast(std::uint16_t, static_cast<_Float16>(x))};
}
template <>
__device__ inline float from_float<float>(float x)
{
    return x;
}

// One call's view of the cache and the batch.
struct Cache {
    std::int8_t* keys;
    std::int8_t* values;
    float* key_scale;
    float* value_scale;
    std::int8_t* bounds;
    unsigned long long* weight;
    std::uint32_t blocks, kv_heads, dim, dims;  // dims: dim rounded up to 64
    std::uint32_t tokens, tile_shift;           // a block's tokens; log2 of its 16-token tiles
};
struct Batch {
    const std::int32_t* table;
    const std::int32_t* lens;
    const std::int32_t* first;  // null: one token of the batch per sequence
    std::uint32_t seqs, width, stride, tokens;
};

// A group of consecutive tokens of one sequence of the batch.  Sequence s owns
// the slots from floor(first[s] / per) + s on, at least one and at least
// ceil(its tokens / per); the host launches floor(tokens / per) + seqs.
struct Group {
    std::uint32_t seq;
    std::int32_t from, count;  // tokens of the sequence's part of the batch
    std::int32_t row;          // batch row of token `from`
    std::int64_t seen;         // tokens of the cache that token `from` attends to
};
// The last of n indices whose base (not decreasing) is not above `value`, 0 if
// there is none.  A wave compares 64 of them at a time, so that up to 64
// sequences cost one trip to memory and 4096 two; all lanes take part.
template <typename F>
__device__ inline std::uint32_t last_not_above(std::uint32_t n, std::uint32_t value, F base)
{
    const std::uint32_t lane = threadIdx.x % kWave;
    std::uint32_t lo = 0;
    while (n > 1) {
        const std::uint32_t step = (n + kWave - 1) / kWave;
        const unsigned long long votes = __ballot(lane * step < n && base(lo + lane * step) <= value);
        const std::uint32_t at = votes == 0 ? 0 : (63 - static_cast<std::uint32_t>(__clzll(static_cast<long long>(votes)))) * step;
        lo += at;
        n = n - at < step ? n - at : step;
        if (votes == 0) break;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}
__device__ inline std::uint32_t slot_base(const Batch& b, std::uint32_t s, std::uint32_t per)
{
    return static_cast<std::uint32_t>(b.first[s]) / per + s;
}
__device__ inline bool find_group(const Batch& b, std::uint32_t slot, std::uint32_t per, Group* g)
{
    std::uint32_t s = slot;
    std::int32_t begin, total;
    if (b.first == nullptr) {
        begin = static_cast<std::int32_t>(slot);
        total = 1;
        g->from = 0;
    } else {
        s = last_not_above(b.seqs, slot, [&](std::uint32_t i) { return slot_base(b, i, per); });
        begin = b.first[s];
        total = b.first[s + 1] - begin;
        const std::uint32_t base = slot_base(b, s, per);
        if (slot < base) {
            return false;
        }
        const std::uint64_t from = static_cast<std::uint64_t>(slot - base) * per;
        if (total <= 0 || from >= static_cast<std::uint64_t>(total)) {
            return false;
        }
        g->from = static_cast<std::int32_t>(from);
    }
    // offsets that do not describe the batch leave their rows out
    if (begin < 0 || static_cast<std::uint64_t>(begin) + total > b.tokens) {
        return false;
    }
    g->seq = s;
    g->count = total - g->from < static_cast<std::int32_t>(per) ? total - g->from
                                                                : static_cast<std::int32_t>(per);
    g->row = begin + g->from;
    g->seen = static_cast<std::int64_t>(b.lens[s]) - total + g->from + 1;
    return true;
}

// A physical block, or -1 for an entry that names none of the pool's.
__device__ inline std::int32_t block_at(const Cache& c, const Batch& b, std::uint32_t seq,
                                        std::int64_t logical)
{
    if (logical < 0 || logical >= static_cast<std::int64_t>(b.width)) {
        return -1;
    }
    const std::int32_t id = b.table[static_cast<std::size_t>(seq) * b.stride + logical];
    return static_cast<std::uint32_t>(id) < c.blocks ? id : -1;
}

// 4 codes -> 4 f16, exactly: 0x6400 | (code + 128) is 1024 + 128 + code.
__device__ inline f16x4 widen(std::uint32_t codes)
{
    const std::uint32_t u = codes ^ 0x80808080u;
    const std::uint32_t a = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    const std::uint32_t b = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    const f16x2 bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    const f16x2 x = __builtin_bit_cast(f16x2, a) - bias, y = __builtin_bit_cast(f16x2, b) - bias;
    return __builtin_shufflevector(x, y, 0, 1, 2, 3);
}
__device__ inline f16x8 widen8(std::uint32_t lo, std::uint32_t hi)
{
    return __builtin_shufflevector(widen(lo), widen(hi), 0, 1, 2, 3, 4, 5, 6, 7);
}

// The larger of three, without the quieting of NaNs that the compiler puts
// before each fmaxf of a value that came through a branch.
__device__ inline float max_of_3(float x, float y, float z)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- attend ---------------------------------------------------------------

struct Attend {
    Cache c;
    Batch b;
    const void* q;
    std::int64_t q_token, q_head;  // strides in elements
    std::uint32_t q_vector;        // rows may be loaded 16 bytes at a time
    std::uint32_t out_vector;      // and stored 8 at a time
    std::uint32_t heads, group;    // query heads; query heads per kv head
    std::uint32_t per;             // tokens per unit
    std::uint32_t row_tiles;       // 16-row tiles per unit (1 unless group > 16)
    std::uint32_t pairs;           // kv heads times row tiles: a unit's workgroups, heads first
    std::uint32_t rows;            // rows of a tile that any unit uses
    std::uint32_t groups;          // units times pairs; a merge's workgroups beyond clear rows
    float scale;                   // softmax scale times log2(e)
    const std::int32_t* selected;
    std::uint32_t count;
    std::uint32_t split, splits;   // tokens per split, splits launched
    void* out;
    float* partial;                // [unit, row tile, kv head, split][rows][dims]
    float* stats;                  // [...][rows][2]: reference exponent, denominator
    float* lse;                    // [tokens, heads], log2 of the row's denominator, or null
    float* tile_sums;              // [unit, row tile, kv head, tile][rows], log2 of a row's sum over a tile
};

// Splits that hold work for a unit whose last token sees `seen` tokens.
__device__ inline std::uint32_t live_splits(const Attend& a, std::int64_t seen)
{
    const std::int64_t n = a.selected != nullptr
                               ? static_cast<std::int64_t>(a.count) * a.c.tokens
                               : seen;
    return seen <= 0 ? 0u : static_cast<std::uint32_t>((n + a.split - 1) / a.split);
}

__device__ inline std::int64_t visible(const Attend& a, std::int64_t seen)
{
    const std::int64_t most = static_cast<std::int64_t>(a.b.width) * a.c.tokens;
    return seen < most ? seen : most;
}

// Four dims of a finished row: sums `o` and denominator `l` at exponent `ref`.
template <typename T>
__device__ inline void finish_row(const Attend& a, std::int64_t token, std::uint32_t head, int d, f32x4 o, float l,
                                  float ref)
{
    T* out = static_cast<T*>(a.out) + (token * a.heads + head) * a.c.dim + d;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    union {
        uint2 v;
        T e[4];
    } u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u.e[i] = from_float<T>(l == 0.0f ? 0.0f : o[i] * inv);
    if ((a.c.dim & 3) == 0 && a.out_vector != 0) {
        if (d < static_cast<int>(a.c.dim)) *reinterpret_cast<uint2*>(out) = u.v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (d + i < static_cast<int>(a.c.dim)) out[i] = u.e[i];
        }
    }
    if (d == 0 && a.lse != nullptr) {
        a.lse[token * a.heads + head] = l == 0.0f ? kInf : ref + log2f(l);
    }
}

// The query rows of a wave as the matrix units take them: lane (quarter, m)
// holds row m's dims 16 quarter .. 16 quarter + 15 of every 64, scaled by a
// power of two; *factor undoes it and applies the softmax scale.
template <typename T, int CH>
__device__ inline void load_query(const Attend& a, std::int64_t token, std::uint32_t head, bool live, int quarter,
                                  f16x8 (&query)[CH * 2], float* factor)
{
    // rows that are not there read the batch's first one and take zeros
    const T* q = static_cast<const T*>(a.q) + (live ? token * a.q_token + head * a.q_head : 0);
    float x[CH * 16];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < CH * 2; ++i) {
        const int d0 = (i / 2) * 64 + quarter * 16 + (i & 1) * 8, dim = static_cast<int>(a.c.dim);
        if (a.q_vector != 0 && dim % 8 == 0) {
            union {
                u32x4 v;
                T e[8];
            } u;
            u.v = *reinterpret_cast<const u32x4*>(q + (d0 < dim ? d0 : 0));
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i * 8 + j] = live && d0 < dim ? to_float(u.e[j]) : 0.0f;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float e = to_float(q[d0 + j < dim ? d0 + j : 0]);
                x[i * 8 + j] = live && d0 + j < dim ? e : 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[i * 8 + j]));
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    // below 2^-46 a row's scores are nothing beside one another's rounding
    int k = top > 0.0f && top < kInf ? 14 - ilogbf(top) : 0;
    k = k > 60 ? 60 : k;
    // the softmax scale's sign goes to the rows, so that the factor is positive
    const float sign = a.scale < 0.0f ? -1.0f : a.scale == 0.0f ? 0.0f : 1.0f;
    *factor = fmaxf(ldexpf(fabsf(a.scale), -k), 0x1p-80f);
#pragma unroll
    for (int i = 0; i < CH * 2; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) query[i][j] = static_cast<_Float16>(ldexpf(sign * x[i * 8 + j], k));
    }
}

// What a wave knows of up to 64 consecutive tiles, one per lane.
struct Tiles {
    std::int32_t id, sub, pos;          // block, tile within it, first token's position
    float key_scale, log_scale, inv_scale;
};

__device__ inline Tiles load_tiles(const Attend& a, std::uint32_t seq, std::uint32_t head, const std::int32_t* list,
                                   std::int64_t tile, bool inside, std::int64_t seen)
{
    Tiles t{0, 0, kNowhere, 0.0f, 0.0f, 1.0f};
    if (inside) {
        const std::int64_t entry = tile >> a.c.tile_shift;
        const std::int64_t logical = list == nullptr ? entry : list[entry];
        const std::int32_t sub = static_cast<std::int32_t>(tile) & ((1 << a.c.tile_shift) - 1);
        const std::int32_t id = block_at(a.c, a.b, seq, logical);
        const std::int64_t pos = logical * a.c.tokens + sub * 16;
        if (id >= 0 && pos < seen) {
            const std::size_t bh = static_cast<std::size_t>(id) * a.c.kv_heads + head;
            float vs = a.c.value_scale[bh];
            const float ks = a.c.key_scale[bh];
            // scales below the least, of blocks not begun yet, have no
            // logarithm or inverse to take part with
            vs = vs < kScaleMin ? kScaleMin : vs;
            // a NaN value scale shows through its logarithm in the rows that
            // see the block, and through nothing in those that do not
            t = Tiles{id, sub, static_cast<std::int32_t>(pos), ks < kScaleMin ? kScaleMin : ks, log2f(vs),
                      vs == vs ? 1.0f / vs : 1.0f};
        }
    }
    return t;
}

__device__ inline std::int32_t lane_int(std::int32_t x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ inline float lane_float(float x, int lane)
{
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// A workgroup of kWaves waves takes one (kv head, row tile, unit; split); its
// waves take a run of 16-token tiles each and join through LDS.  A lane looks
// up one tile of the wave's next 64 (block, scales), so the loop itself has no
// dependent loads; the keys of the pair of tiles after this one are on their
// way while its softmax runs, the values while the next scores do.
// It reads the codes once and is bound by HBM: 64 sequences of 1024..32768
// tokens (2.44 GB) in 424 us, 5.75 TB/s; one of 262,147 (0.54 GB) in 89 us,
// 6.07 TB/s (a sum over 4 GiB reaches 6.14 here, a copy 4.79 read and
// written).  16 rows of a product serve 1 to 16 query rows alike, since the
// matrix units are idle otherwise.
// kWeigh: each tile's sum of a row's weights is left behind as one logarithm,
// from which k_kv_weigh makes probabilities once the row's denominator is known.
// kOnce: a sequence's codes have one unit of rows in the step, whose workgroups
// read them once, past the caches as streams do (6.1 against 5.4 TB/s over one
// sequence of 262,147 tokens; 422 against 467 us over 64 of 1024..32768).
template <typename T, int CH, int kWaves, bool kWeigh, bool kOnce>
__global__ __launch_bounds__(kWaves * kWave, CH <= 2 ? 4 : CH == 3 ? 2 : 1) void k_kv_attend(Attend a)
{
    constexpr int P = CH * 64, kRow = P + 4;
    extern __shared__ float s_out[];  // [kWaves][rows][kRow]
    __shared__ float s_ref[kWaves][16], s_den[kWaves][16];

    const std::uint32_t unit = blockIdx.x / a.pairs, pair = blockIdx.x % a.pairs;
    const std::uint32_t head = pair % a.c.kv_heads, row_tile = pair / a.c.kv_heads;
    const std::uint32_t split = blockIdx.y;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int m = lane & 15, quarter = lane >> 4;

    Group g;
    if (!find_group(a.b, unit, a.per, &g)) {
        return;
    }
    const std::int64_t seen = visible(a, g.seen + g.count - 1);
    const std::uint32_t live = live_splits(a, seen);
    if (split >= live && !(split == 0 && a.splits == 1)) {
        return;
    }

    // this lane's query row
    const std::uint32_t r = row_tile * 16 + m;
    const std::uint32_t row_token = r / a.group, row_head = r % a.group;
    const bool row_live = row_token < static_cast<std::uint32_t>(g.count);
    const std::int64_t limit64 = row_live ? visible(a, g.seen + row_token) : 0;
    const int limit = limit64 > 0 ? static_cast<int>(limit64) : 0;
    const std::int64_t token_row = g.row + static_cast<std::int64_t>(row_token);

    f16x8 query[CH * 2];
    float factor;
    load_query<T, CH>(a, token_row, head * a.group + row_head, row_live, quarter, query, &factor);

    f32x4 acc[CH * 4];
#pragma unroll
    for (int i = 0; i < CH * 4; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float ref = kLowest, den = 0.0f;

    const std::int64_t total = a.selected != nullptr ? static_cast<std::int64_t>(a.count) * a.c.tokens : seen;
    const std::int64_t begin = static_cast<std::int64_t>(split) * a.split;
    const std::int64_t end = begin + a.split < total ? begin + a.split : total;
    const std::int32_t* list =
        a.selected == nullptr ? nullptr
                              : a.selected + (static_cast<std::int64_t>(g.row) * a.c.kv_heads + head) * a.count;
    const std::size_t head_bytes = static_cast<std::size_t>(a.c.tokens) * P;
    float* sums = kWeigh ? a.tile_sums + (static_cast<std::size_t>(blockIdx.x) * a.c.tokens / 16 * a.b.width + begin / 16) * a.rows
                         : nullptr;
    const std::int64_t tiles = end > begin ? (end - begin + 15) / 16 : 0;
    const std::int64_t per_wave = (tiles + 2 * kWaves - 1) / (2 * kWaves) * 2;
    const std::int64_t tile0 = wave * per_wave;
    const std::int64_t tile1 = tile0 + per_wave < tiles ? tile0 + per_wave : tiles;

    for (std::int64_t at = tile0; at < tile1; at += kWave) {
        const int n = static_cast<int>(tile1 - at < kWave ? tile1 - at : kWave);
        const Tiles info = load_tiles(a, g.seq, head, list, begin / 16 + at + lane, lane < n, seen);
        u32x4 kc[2][CH], vc[2][CH];
        const auto tile_at = [&](const std::int8_t* pool, int tile) {
            const std::size_t bh = static_cast<std::size_t>(lane_int(info.id, tile)) * a.c.kv_heads + head;
            return reinterpret_cast<const u32x4*>(pool + bh * head_bytes +
                                                  static_cast<std::size_t>(lane_int(info.sub, tile)) * 16 * P);
        };
        const auto load = [&](u32x4 (&to)[2][CH], const std::int8_t* pool, int tile) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const u32x4* p = tile_at(pool, tile + u);
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    to[u][i] = kOnce ? __builtin_nontemporal_load(p + i * kWave + lane) : p[i * kWave + lane];
                }
            }
        };
        const auto step = [&](int tile, bool more) __attribute__((always_inline)) {
            f32x4 s[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8(kc[u][i].x, kc[u][i].y), query[2 * i], s[u], 0, 0, 0);
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8(kc[u][i].z, kc[u][i].w), query[2 * i + 1], s[u], 0, 0, 0);
                }
            }
            if (more) load(kc, a.c.keys, tile + 2);
            float t[2][4];
            float top = -kInf;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float f = factor * lane_float(info.key_scale, tile + u), e = lane_float(info.log_scale, tile + u);
                const int left = limit - lane_int(info.pos, tile + u) - quarter * 4;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    t[u][i] = i < left ? fmaf(s[u][i], f, e) : -kInf;
                    top = fmaxf(top, t[u][i]);
                }
            }
            // The row's reference exponent stays 2^7 to 2^15 below its largest
            // weight (the f16 range), so it moves only now and then.
            if (__any(top > ref + 15.0f)) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float next = fmaxf(ref, top - 7.0f);
                const float shrink = exp2_fast(ref - next);
                ref = next;
                den *= shrink;
#pragma unroll
                for (int i = 0; i < CH * 4; ++i) acc[i] *= shrink;
            }
            f16x8 w;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = exp2_fast(t[u][i] - ref);
                    sum += x;
                    w[u * 4 + i] = static_cast<_Float16>(x);
                }
                const float part = sum * lane_float(info.inv_scale, tile + u);
                den += part;
                if (kWeigh) {
                    float all = part + __shfl_xor(part, 16);
                    all += __shfl_xor(all, 32);
                    if (quarter == 0 && m < static_cast<int>(a.rows) && tile + u < n) {
                        sums[(at + tile + u) * a.rows + m] = __builtin_amdgcn_logf(all) + ref;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < CH; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[i * 4 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8(vc[0][i][j], vc[1][i][j]), w,
                                                                            acc[i * 4 + j], 0, 0, 0);
                }
            }
            if (more) load(vc, a.c.values, tile + 2);
        };
        load(kc, a.c.keys, 0);
        load(vc, a.c.values, 0);
        int tile = 0;
        for (; tile + 2 < n; tile += 2) step(tile, true);
        step(tile, false);
    }
    den += __shfl_xor(den, 16);
    den += __shfl_xor(den, 32);

    if (quarter == 0) {
        s_ref[wave][m] = ref;
        s_den[wave][m] = den;
    }
    __syncthreads();
    float top = s_ref[0][m];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) top = fmaxf(top, s_ref[i][m]);
    const float mine = exp2_fast(ref - top);
    const int rows = static_cast<int>(a.rows);
    if (m < rows) {
#pragma unroll
        for (int i = 0; i < CH * 4; ++i) {
            *reinterpret_cast<f32x4*>(&s_out[(wave * rows + m) * kRow + i * 16 + quarter * 4]) = acc[i] * mine;
        }
    }
    __syncthreads();

    const std::uint32_t unit_rows = g.count * a.group;
    for (int i = threadIdx.x; i < rows * (P / 4); i += kWaves * kWave) {
        const int row = i / (P / 4), d = i % (P / 4) * 4;
        const std::uint32_t rr = row_tile * 16 + row;
        if (rr >= unit_rows) {
            continue;
        }
        float top_row = s_ref[0][row];
#pragma unroll
        for (int k = 1; k < kWaves; ++k) top_row = fmaxf(top_row, s_ref[k][row]);
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            o += *reinterpret_cast<const f32x4*>(&s_out[(k * rows + row) * kRow + d]);
            l = fmaf(s_den[k][row], exp2_fast(s_ref[k][row] - top_row), l);
        }
        if (a.splits == 1) {
            finish_row<T>(a, g.row + static_cast<std::int64_t>(rr / a.group), head * a.group + rr % a.group, d, o, l,
                          top_row);
        } else {
            const std::size_t cell =
                (static_cast<std::size_t>(blockIdx.x) * a.splits + split) * rows + row;
            *reinterpret_cast<f32x4*>(&a.partial[cell * P + d]) = o;
            if (d == 0) {
                a.stats[cell * 2] = top_row;
                a.stats[cell * 2 + 1] = l;
            }
        }
    }
}

// attend for chunks of many tokens, where the matrix units and the softmax's
// vector work bound it and not memory.  A workgroup of four waves takes
// 4 * RT * 16 query rows of one kv head (consecutive tokens, every head of the
// group) and one split; the waves share the cache's tiles, which they widen to
// f16 once for all of them and keep in LDS in lane order (a 16-byte read per
// lane per operand, free of conflicts, two buffers), and each keeps RT tiles of
// 16 rows in registers, so that an operand read serves RT products.
// 16 chunks of 2,048 tokens over 16,384 (8.2e12 operations) take 8.1-8.5 ms by
// card, about 1,000 TFLOP/s (a large library product reaches 1,420 here); two
// chunks of about 2,000 over 12,001..16,384 take 1.08-1.16 ms, the last of two
// rounds of workgroups partly empty.  8 of 1,024 over 8,192 take 3.55 ms at 256
// dims and 1.95 at 192, where accumulators leave room for one and two row tiles
// and an operand read serves as few products.  At 128 dims the matrix units are
// busy 43 % of the time, the vector units 59 %: 180 vector instructions a pair
// of tiles (24 exponentials; scale, maximum, sum and rounding of 24 scores a
// lane; widening) beside 48 products, and vector work runs at half rate while
// the matrix unit of its SIMD does, so that their sum bounds it more than either.
template <typename T, int CH, int RT>
__global__ __launch_bounds__(256, 2) void k_kv_attend_many(Attend a)
{
    constexpr int P = CH * 64;
    constexpr int kTiles = CH <= 2 ? 4 : 2;            // 16-token tiles per stage
    constexpr int kKeys = kTiles * CH, kValues = kTiles / 2 * CH;
    constexpr int kKeysEach = (kKeys + 3) / 4, kValuesEach = (kValues + 3) / 4;
    constexpr int kKeyBytes = kTiles * CH * 2048, kStage = 2 * kKeyBytes;
    extern __shared__ unsigned char s_stage[];        // [2][kStage]: keys, then values

    const std::uint32_t split = blockIdx.y;
    // the last tokens of a chunk see the most: they start first
    const std::uint32_t block = gridDim.x - 1 - blockIdx.x;
    const std::uint32_t unit = block / a.pairs, head = block % a.pairs;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int m = lane & 15, quarter = lane >> 4;

    Group g;
    if (!find_group(a.b, unit, a.per, &g)) {
        return;
    }
    const std::int64_t seen = visible(a, g.seen + g.count - 1);
    const std::uint32_t live = live_splits(a, seen);
    if (split >= live && !(split == 0 && a.splits == 1)) {
        return;
    }

    f16x8 query[RT][CH * 2];
    float factor[RT], ref[RT], den[RT], over[RT];  // over: how far a score may pass ref
    int limit[RT];
    int least = 0x7fffffff;  // tokens that every row of the wave sees
    f32x4 acc[RT][CH * 4];
#pragma unroll
    for (int k = 0; k < RT; ++k) {
        const std::uint32_t r = (wave * RT + k) * 16 + m;
        const std::uint32_t row_token = r / a.group, row_head = r % a.group;
        const bool row_live = row_token < static_cast<std::uint32_t>(g.count);
        const std::int64_t limit64 = row_live ? visible(a, g.seen + row_token) : 0;
        limit[k] = limit64 > 0 ? static_cast<int>(limit64) : 0;
        least = row_live && limit[k] < least ? limit[k] : least;
        load_query<T, CH>(a, g.row + static_cast<std::int64_t>(row_token), head * a.group + row_head, row_live, quarter,
                          query[k], &factor[k]);
        ref[k] = 0.0f;
        den[k] = 0.0f;
        over[k] = kLowest;
#pragma unroll
        for (int i = 0; i < CH * 4; ++i) acc[k][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) {
        const int x = __shfl_xor(least, k);
        least = x < least ? x : least;
    }
    least = __builtin_amdgcn_readfirstlane(least);

    const std::int64_t begin = static_cast<std::int64_t>(split) * a.split;
    const std::int64_t end = begin + a.split < seen ? begin + a.split : seen;
    const std::int64_t tiles = end > begin ? (end - begin + 15) / 16 : 0;
    const std::int64_t stages = (tiles + kTiles - 1) / kTiles;
    const std::size_t head_bytes = static_cast<std::size_t>(a.c.tokens) * P;

    Tiles info, seen_info;  // of the stages being fetched, and of those being computed
    u32x4 kreg[kKeysEach], vreg[kValuesEach][2];
    const auto look_up = [&](std::int64_t stage) {  // the 64 tiles from this stage on
        const std::int64_t at = stage * kTiles + lane;
        info = load_tiles(a, g.seq, head, nullptr, begin / 16 + at, at < tiles, seen);
    };
    const auto tile_at = [&](const std::int8_t* pool, int tile) {
        const std::size_t bh = static_cast<std::size_t>(lane_int(info.id, tile)) * a.c.kv_heads + head;
        return reinterpret_cast<const u32x4*>(pool + bh * head_bytes +
                                              static_cast<std::size_t>(lane_int(info.sub, tile)) * 16 * P);
    };
    const auto fetch = [&](std::int64_t stage) {
        const int t0 = static_cast<int>(stage % (kWave / kTiles)) * kTiles;
#pragma unroll
        for (int k = 0; k < kKeysEach; ++k) {
            const int u = wave + 4 * k;
            if (u < kKeys) kreg[k] = tile_at(a.c.keys, t0 + u / CH)[u % CH * kWave + lane];
        }
#pragma unroll
        for (int k = 0; k < kValuesEach; ++k) {
            const int u = wave + 4 * k;
            if (u < kValues) {
                vreg[k][0] = tile_at(a.c.values, t0 + u / CH * 2)[u % CH * kWave + lane];
                vreg[k][1] = tile_at(a.c.values, t0 + u / CH * 2 + 1)[u % CH * kWave + lane];
            }
        }
    };
    const auto put = [&](std::int64_t stage) {
        f16x8* keys = reinterpret_cast<f16x8*>(s_stage + (stage & 1) * kStage);
        f16x8* values = keys + kKeyBytes / 16;
#pragma unroll
        for (int k = 0; k < kKeysEach; ++k) {
            const int u = wave + 4 * k;
            if (u < kKeys) {
                keys[(2 * u) * kWave + lane] = widen8(kreg[k].x, kreg[k].y);
                keys[(2 * u + 1) * kWave + lane] = widen8(kreg[k].z, kreg[k].w);
            }
        }
#pragma unroll
        for (int k = 0; k < kValuesEach; ++k) {
            const int u = wave + 4 * k;
            if (u < kValues) {
#pragma unroll
                for (int j = 0; j < 4; ++j) values[(4 * u + j) * kWave + lane] = widen8(vreg[k][0][j], vreg[k][1][j]);
            }
        }
    };
    const auto compute = [&](std::int64_t stage) __attribute__((always_inline)) {
        const int t0 = static_cast<int>(stage % (kWave / kTiles)) * kTiles;
        const f16x8* keys = reinterpret_cast<const f16x8*>(s_stage + (stage & 1) * kStage) + lane;
        const f16x8* values = keys + kKeyBytes / 16;
#pragma unroll 1
        for (int tile = t0; tile < t0 + kTiles; tile += 2) {
            f32x4 s[2][RT];
            float f[2], e[2];
            int pos[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                pos[u] = lane_int(seen_info.pos, tile + u);
                f[u] = lane_float(seen_info.key_scale, tile + u);
                e[u] = lane_float(seen_info.log_scale, tile + u);
#pragma unroll
                for (int k = 0; k < RT; ++k) s[u][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < CH * 2; ++i) {
                    const f16x8 key = keys[(u * CH * 2 + i) * kWave];
#pragma unroll
                    for (int k = 0; k < RT; ++k) s[u][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, query[k][i], s[u][k], 0, 0, 0);
                }
            }
            const bool whole = (pos[0] > pos[1] ? pos[0] : pos[1]) + 16 <= least;
            // scores as exponents above the row's reference
#pragma unroll
            for (int k = 0; k < RT; ++k) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float scale = factor[k] * f[u], shift = e[u] - ref[k];
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[u][k][i] = fmaf(s[u][k][i], scale, shift);
                }
            }
            if (!whole) {
#pragma unroll
                for (int k = 0; k < RT; ++k) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int left = limit[k] - pos[u] - quarter * 4;
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[u][k][i] = i < left ? s[u][k][i] : -kInf;
                    }
                }
            }
            float top[RT];
            bool move = false;
#pragma unroll
            for (int k = 0; k < RT; ++k) {
                top[k] = max_of_3(s[0][k][0], s[0][k][1], max_of_3(s[0][k][2], s[0][k][3], max_of_3(s[1][k][0], s[1][k][1], max_of_3(s[1][k][2], s[1][k][3], s[1][k][3]))));
                move |= top[k] > over[k];
            }
            if (__any(move)) {
#pragma unroll
                for (int k = 0; k < RT; ++k) {
                    float t = fmaxf(top[k], __shfl_xor(top[k], 16));
                    t = fmaxf(t, __shfl_xor(t, 32));
                    // up for a row that has sums, either way for one that has none
                    const float up = t > over[k] ? t - 7.0f : 0.0f;
                    const float shrink = over[k] == kLowest ? 0.0f : exp2_fast(-up);
                    over[k] = t > over[k] ? 15.0f : over[k];
                    ref[k] += up;
                    den[k] *= shrink;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[u][k][i] -= up;
                    }
#pragma unroll
                    for (int i = 0; i < CH * 4; ++i) acc[k][i] *= shrink;
                }
            }
            f16x8 w[RT];
#pragma unroll
            for (int k = 0; k < RT; ++k) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = exp2_fast(s[u][k][i]);
                        w[k][u * 4 + i] = static_cast<_Float16>(x[i]);
                    }
                    // The f32 weights, not the rounded ones that the products take: in a block
                    // of a small value scale these lose bits or vanish, and with them the
                    // block's whole share, since inv_scale brings the sum back up.
                    const float sum = (x[0] + x[1]) + (x[2] + x[3]);
                    den[k] = fmaf(sum, lane_float(seen_info.inv_scale, tile + u), den[k]);
                }
            }
#pragma unroll
            for (int i = 0; i < CH * 4; ++i) {
                const f16x8 value = values[i * kWave];
#pragma unroll
                for (int k = 0; k < RT; ++k) acc[k][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value, w[k], acc[k][i], 0, 0, 0);
            }
            keys += CH * 4 * kWave;
            values += CH * 4 * kWave;
        }
    };
    if (stages > 0) {
        look_up(0);
        fetch(0);
        put(0);
        if (stages > 1) fetch(1);
        seen_info = info;
    }
    __syncthreads();
    for (std::int64_t stage = 0; stage < stages; ++stage) {
        if (stage % (kWave / kTiles) == 0) seen_info = info;
        if (stage + 1 < stages) put(stage + 1);
        if (stage + 2 < stages) {
            if ((stage + 2) % (kWave / kTiles) == 0) look_up(stage + 2);
            fetch(stage + 2);
        }
        compute(stage);
        __syncthreads();
    }

#pragma unroll
    for (int k = 0; k < RT; ++k) {
        den[k] += __shfl_xor(den[k], 16);
        den[k] += __shfl_xor(den[k], 32);
        const std::uint32_t r = (wave * RT + k) * 16 + m;
        if (r >= g.count * a.group) {
            continue;
        }
        if (a.splits == 1) {
            const std::int64_t token = g.row + static_cast<std::int64_t>(r / a.group);
            const std::uint32_t h = head * a.group + r % a.group;
#pragma unroll
            for (int i = 0; i < CH * 4; ++i) finish_row<T>(a, token, h, i * 16 + quarter * 4, acc[k][i], den[k], ref[k]);
        } else {
            const std::size_t cell = (static_cast<std::size_t>(block) * a.splits + split) * a.rows + r;
#pragma unroll
            for (int i = 0; i < CH * 4; ++i) {
                *reinterpret_cast<f32x4*>(&a.partial[cell * P + i * 16 + quarter * 4]) = acc[k][i];
            }
            if (quarter == 0) {
                a.stats[cell * 2] = over[k] == kLowest ? kLowest : ref[k];
                a.stats[cell * 2 + 1] = den[k];
            }
        }
    }
}

// Zeros in the step's rows that belong to no sequence: before the first one's,
// from the last one's end on, or of one that ends past the step.  The merge
// does it in workgroups behind its own, k_kv_clear_rest where there is no merge
// (2 us of a call).  Within the attention's kernels the same lines cost registers:
// 3.54 -> 4.44 ms for 8 chunks of 1,024 tokens over 8,192 at 256 dims.
template <typename T>
__device__ inline void clear_rest(const Attend& a, std::uint32_t at, std::uint32_t each)
{
    const std::int64_t tokens = a.b.tokens;
    std::int64_t lo = a.b.first[0], hi = a.b.first[a.b.seqs];
    if (hi > tokens) {
        hi = a.b.first[last_not_above(a.b.seqs + 1, a.b.tokens, [&](std::uint32_t i) {
            return static_cast<std::uint32_t>(a.b.first[i]);
        })];
    }
    lo = lo < 0 ? 0 : lo < tokens ? lo : tokens;
    hi = hi < lo ? lo : hi < tokens ? hi : tokens;
    const std::int64_t wide = static_cast<std::int64_t>(a.heads) * a.c.dim;
    for (std::int64_t i = at; i < lo + tokens - hi; i += each) {
        T* out = static_cast<T*>(a.out) + (i < lo ? i : hi + (i - lo)) * wide;
        for (std::int64_t e = threadIdx.x; e < wide; e += 256) out[e] = T{};
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_kv_clear_rest(Attend a)
{
    clear_rest<T>(a, blockIdx.x, gridDim.x);
}

// Joins a unit's splits where there are few of them: a thread takes four dims
// of a row and goes through the splits, a workgroup as many rows as fit.
template <typename T>
__global__ __launch_bounds__(256) void k_kv_merge_few(Attend a)
{
    if (blockIdx.x >= a.groups) {
        if (blockIdx.y == 0) clear_rest<T>(a, blockIdx.x - a.groups, gridDim.x - a.groups);
        return;
    }
    const std::uint32_t unit = blockIdx.x / a.pairs, pair = blockIdx.x % a.pairs;
    const std::uint32_t head = pair % a.c.kv_heads, row_tile = pair / a.c.kv_heads;
    const std::uint32_t quads = a.c.dims / 4, groups = 256 / quads;
    const std::uint32_t row = blockIdx.y * groups + threadIdx.x / quads, d = threadIdx.x % quads * 4;
    Group g;
    if (!find_group(a.b, unit, a.per, &g)) {
        return;
    }
    const std::uint32_t rr = row_tile * 16 + row;
    if (threadIdx.x >= groups * quads || row >= a.rows || rr >= g.count * a.group) {
        return;
    }
    const int live = static_cast<int>(live_splits(a, visible(a, g.seen + g.count - 1)));
    const std::size_t cell0 = static_cast<std::size_t>(blockIdx.x) * a.splits * a.rows + row;
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + cell0;
    const float* partial = a.partial + cell0 * a.c.dims + d;
    float top = kLowest;
    for (int s = 0; s < live; ++s) top = fmaxf(top, stats[static_cast<std::size_t>(s) * a.rows].x);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll 4
    for (int s = 0; s < live; ++s) {
        const float2 x = stats[static_cast<std::size_t>(s) * a.rows];
        const float f = exp2_fast(x.x - top);
        o += *reinterpret_cast<const f32x4*>(partial + static_cast<std::size_t>(s) * a.rows * a.c.dims) * f;
        l = fmaf(x.y, f, l);
    }
    finish_row<T>(a, g.row + static_cast<std::int64_t>(rr / a.group), head * a.group + rr % a.group, static_cast<int>(d),
                  o, l, top);
}

// Joins a unit's splits: one workgroup per (kv head, row tile; unit; row).
// Its threads first turn the splits' reference exponents into factors, then
// take dims in fours and the splits in turn.
template <typename T>
__global__ __launch_bounds__(256) void k_kv_merge(Attend a)
{
    constexpr int kChunk = 256;
    __shared__ float s_factor[kChunk], s_wave[4], s_sum[4];
    __shared__ f32x4 s_part[256];
    if (blockIdx.x >= a.groups) {
        if (blockIdx.y == 0) clear_rest<T>(a, blockIdx.x - a.groups, gridDim.x - a.groups);
        return;
    }
    const std::uint32_t unit = blockIdx.x / a.pairs, pair = blockIdx.x % a.pairs, row = blockIdx.y;
    const std::uint32_t head = pair % a.c.kv_heads, row_tile = pair / a.c.kv_heads;
    const int P = static_cast<int>(a.c.dims), lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    Group g;
    if (!find_group(a.b, unit, a.per, &g)) {
        return;
    }
    const std::uint32_t rr = row_tile * 16 + row;  // row tiles are whole where there are several
    if (rr >= g.count * a.group) {
        return;
    }
    const int live = static_cast<int>(live_splits(a, visible(a, g.seen + g.count - 1)));
    const std::size_t cell0 = static_cast<std::size_t>(blockIdx.x) * a.splits * a.rows + row;
    const float2* stats = reinterpret_cast<const float2*>(a.stats);
    float top = kLowest;
    for (int s = threadIdx.x; s < live; s += 256) top = fmaxf(top, stats[cell0 + static_cast<std::size_t>(s) * a.rows].x);
    for (int k = 1; k < kWave; k *= 2) top = fmaxf(top, __shfl_xor(top, k));
    if (lane == 0) s_wave[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_wave[0], s_wave[1]), fmaxf(s_wave[2], s_wave[3]));

    const int quads = P / 4, groups = 256 / quads;  // threads that share a quad of dims
    const int d = threadIdx.x % quads * 4, part = threadIdx.x / quads;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
    for (int s0 = 0; s0 < live; s0 += kChunk) {
        const int s = s0 + static_cast<int>(threadIdx.x);
        float f = 0.0f;
        if (s < live) {
            const float2 x = stats[cell0 + static_cast<std::size_t>(s) * a.rows];
            f = exp2_fast(x.x - top);
            l = fmaf(x.y, f, l);
        }
        __syncthreads();
        s_factor[threadIdx.x] = f;
        __syncthreads();
        if (part < groups) {
            const int n = live - s0 < kChunk ? live - s0 : kChunk;
#pragma unroll 4
            for (int k = part; k < n; k += groups) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(
                    &a.partial[(cell0 + static_cast<std::size_t>(s0 + k) * a.rows) * P + d]);
                o += x * s_factor[k];
            }
        }
    }
    for (int k = 1; k < kWave; k *= 2) l += __shfl_xor(l, k);
    if (lane == 0) s_sum[wave] = l;
    s_part[threadIdx.x] = o;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < quads) {
        for (int k = 1; k < groups; ++k) o += s_part[threadIdx.x + k * quads];
        finish_row<T>(a, g.row + static_cast<std::int64_t>(rr / a.group), head * a.group + rr % a.group, d, o,
                      s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3], top);
    }
}

// What a lane's row (m of the unit's row tile) divides its weights by, as a
// logarithm; infinite for a row that adds none: one that is not there or sees
// nothing, and those of a token any of whose heads in the group is not a
// number.  A whole token is left out, whichever rows share its unit or tile.
// All lanes of a wave call it, m from lane & 15.
__device__ inline float weigh_lse(const Attend& a, const Group& g, std::uint32_t head, std::uint32_t row_tile)
{
    const std::uint32_t m = threadIdx.x & 15, r = row_tile * 16 + m;
    const float* lse = a.lse + g.row * static_cast<std::int64_t>(a.heads) + head * a.group;
    const bool there = r < g.count * a.group && m < a.rows;
    const float l = there ? lse[static_cast<std::int64_t>(r / a.group) * a.heads + r % a.group] : kInf;
    bool lost;
    if (a.row_tiles > 1) {  // one token a unit, its heads in several tiles
        bool bad = false;
        for (std::uint32_t h = threadIdx.x % kWave; h < a.group; h += kWave) bad |= lse[h] != lse[h];
        lost = __any(bad);
    } else {
        const std::uint32_t votes = static_cast<std::uint32_t>(__ballot(l != l)) & 0xffffu;
        lost = (votes >> (m / a.group * a.group) & ((1u << a.group) - 1)) != 0;
    }
    return lost ? kInf : l;
}

// weight[block, head] += the probabilities of the unit's rows over the block,
// from the tiles' sums: one thread per block.  Sums are f32 within a block and
// joined as integers, so the order in which blocks of shared prefixes are
// reached does not change them.  24 sequences of 777..20,001 tokens: 7.5 us.
__device__ inline void add_weight(const Attend& a, std::size_t bh, float sum)
{
    if (sum < 1e9f) {  // rows that are not numbers are left out before
        atomicAdd(a.c.weight + bh, static_cast<unsigned long long>(__double2ull_rn(static_cast<double>(sum) * 0x1p32)));
    }
}

__global__ __launch_bounds__(256) void k_kv_weigh(Attend a)
{
    __shared__ float s_lse[16];
    const std::uint32_t unit = blockIdx.x / a.pairs, pair = blockIdx.x % a.pairs;
    const std::uint32_t head = pair % a.c.kv_heads, row_tile = pair / a.c.kv_heads;
    Group g;
    if (!find_group(a.b, unit, a.per, &g)) {
        return;
    }
    const std::int64_t seen = visible(a, g.seen + g.count - 1);
    if (seen <= 0 || static_cast<std::int64_t>(blockIdx.y) * 256 * a.c.tokens >= seen) {
        return;
    }
    if (threadIdx.x < kWave) {
        const float l = weigh_lse(a, g, head, row_tile);
        if (threadIdx.x < a.rows) s_lse[threadIdx.x] = l;
    }
    __syncthreads();
    const std::uint32_t blk = blockIdx.y * 256 + threadIdx.x;
    const std::int32_t id = static_cast<std::int64_t>(blk) * a.c.tokens < seen ? block_at(a.c, a.b, g.seq, blk) : -1;
    if (id < 0) {
        return;
    }
    const std::uint32_t per_block = a.c.tokens / 16;
    const float* sums = a.tile_sums + (static_cast<std::size_t>(blockIdx.x) * a.b.width + blk) * per_block * a.rows;
    float sum = 0.0f;
    for (std::uint32_t tile = 0; tile < per_block && (static_cast<std::int64_t>(blk) * per_block + tile) * 16 < seen; ++tile) {
        for (std::uint32_t k = 0; k < a.rows; ++k) {
            const float l = s_lse[k];
            sum += l == kInf ? 0.0f : exp2_fast(sums[tile * a.rows + k] - l);
        }
    }
    add_weight(a, static_cast<std::size_t>(id) * a.c.kv_heads + head, sum);
}

// The same where the many-row form ran, from the keys again: one wave per
// block of the sequence; 16 query rows at a time, so that every 16 rows widen
// the keys anew and this takes longer than the attention itself: 2 chunks of
// 2,048 tokens over 16,384 (8 kv heads, D = 128) 2.33 ms beside 1.13 + 0.04.
template <typename T, int CH>
__global__ __launch_bounds__(256) void k_kv_weigh_again(Attend a)
{
    constexpr int P = CH * 64;
    const std::uint32_t unit = blockIdx.x / a.pairs, pair = blockIdx.x % a.pairs;
    const std::uint32_t head = pair % a.c.kv_heads, row_tile = pair / a.c.kv_heads;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int m = lane & 15, quarter = lane >> 4;
    Group g;
    if (!find_group(a.b, unit, a.per, &g)) {
        return;
    }
    const std::int64_t seen = visible(a, g.seen + g.count - 1);
    if (seen <= 0) {
        return;
    }
    const std::uint32_t r = row_tile * 16 + m;
    const std::uint32_t row_token = r / a.group, row_head = r % a.group;
    const float lse = weigh_lse(a, g, head, row_tile);
    const bool row_live = lse != kInf;
    const std::int64_t limit64 = row_live ? visible(a, g.seen + row_token) : 0;
    const int limit = limit64 > 0 ? static_cast<int>(limit64) : 0;
    const std::int64_t token_row = g.row + static_cast<std::int64_t>(row_token);
    f16x8 query[CH * 2];
    float factor;
    load_query<T, CH>(a, token_row, head * a.group + row_head, row_live, quarter, query, &factor);
    const std::size_t head_bytes = static_cast<std::size_t>(a.c.tokens) * P;
    const std::uint32_t nb = static_cast<std::uint32_t>((seen + a.c.tokens - 1) / a.c.tokens);
    for (std::uint32_t blk = blockIdx.y * 4 + wave; blk < nb; blk += gridDim.y * 4) {
        const std::int32_t id = block_at(a.c, a.b, g.seq, blk);
        if (id < 0) {
            continue;
        }
        const std::size_t bh = static_cast<std::size_t>(id) * a.c.kv_heads + head;
        const float f = factor * a.c.key_scale[bh];
        float sum = 0.0f;
        for (std::uint32_t sub = 0; sub < a.c.tokens / 16; ++sub) {
            const u32x4* kp = reinterpret_cast<const u32x4*>(a.c.keys + bh * head_bytes +
                                                             static_cast<std::size_t>(sub) * 16 * P);
            f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const u32x4 k = kp[i * kWave + lane];
                s = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8(k.x, k.y), query[2 * i], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8(k.z, k.w), query[2 * i + 1], s, 0, 0, 0);
            }
            const std::int64_t pos = static_cast<std::int64_t>(blk) * a.c.tokens + sub * 16 + quarter * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sum += pos + i < limit ? exp2_fast(fmaf(s[i], f, -lse)) : 0.0f;
            }
        }
#pragma unroll
        for (int x = 1; x < kWave; x *= 2) sum += __shfl_xor(sum, x);
        if (lane == 0) {
            add_weight(a, bh, sum);
        }
    }
}

// ---- append and read ------------------------------------------------------

struct Append {
    Cache c;
    Batch b;
    const void* x[2];                       // keys, values
    std::int64_t token_stride[2], head_stride[2];
    std::uint32_t vector[2];                // rows may be loaded 16 bytes at a time
};

__device__ inline float quantise(float x, float inv)
{
    const float r = rintf(x * inv);
    return r != r ? 0.0f : fminf(fmaxf(r, -127.0f), 127.0f);
}

// The block `slot` of the batch's writes and the new tokens in it.
struct Write {
    std::int32_t id;
    int begin, end;       // the block's slots that get new tokens
    std::int64_t row;     // batch row of slot `begin`
};
__device__ inline bool find_write(const Append& a, std::uint32_t slot, Write* w)
{
    const std::uint32_t t = a.c.tokens;
    std::uint32_t s = slot;
    std::int32_t begin = static_cast<std::int32_t>(slot), total = 1;
    std::uint64_t nth = 0;
    if (a.b.first != nullptr) {
        // sequence s owns the slots from floor(first[s] / t) + 2 s on
        const auto base = [&](std::uint32_t i) {
            return static_cast<std::uint32_t>(a.b.first[i]) / t + 2 * i;
        };
        s = last_not_above(a.b.seqs, slot, base);
        if (slot < base(s)) {
            return false;
        }
        begin = a.b.first[s];
        total = a.b.first[s + 1] - begin;
        nth = slot - base(s);
    }
    if (total <= 0 || begin < 0 || static_cast<std::uint64_t>(begin) + total > a.b.tokens) {
        return false;
    }
    const std::int64_t from = static_cast<std::int64_t>(a.b.lens[s]) - total, to = from + total;
    if (from < 0) {
        return false;
    }
    const std::int64_t blk = from / t + static_cast<std::int64_t>(nth);
    if (blk * t >= to) {
        return false;
    }
    w->id = block_at(a.c, a.b, s, blk);
    if (w->id < 0) {
        return false;
    }
    w->begin = from > blk * t ? static_cast<int>(from - blk * t) : 0;
    w->end = to < (blk + 1) * t ? static_cast<int>(to - blk * t) : static_cast<int>(t);
    w->row = begin + (blk * t + w->begin - from);
    return true;
}

// 16 consecutive elements of a row from d0 on, zeros past its dim.
template <typename T>
__device__ inline void load_16(const T* row, int d0, int dim, bool vector, float (&x)[16])
{
    constexpr int kEach = 16 / sizeof(T);
    if (vector && dim % kEach == 0) {
#pragma unroll
        for (int i = 0; i < 16; i += kEach) {
            union {
                u32x4 v;
                T e[kEach];
            } u;
            u.v = *reinterpret_cast<const u32x4*>(row + (d0 + i < dim ? d0 + i : 0));
#pragma unroll
            for (int j = 0; j < kEach; ++j) x[i + j] = d0 + i < dim ? to_float(u.e[j]) : 0.0f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float e = to_float(row[d0 + i < dim ? d0 + i : 0]);
            x[i] = d0 + i < dim ? e : 0.0f;
        }
    }
}

// rint(x * inv) of four values as bytes.  Adding 1.5 * 2^23 leaves the whole
// number nearest to the rounded product in the low bits, so the two must not
// become one fused step; it needs no limit, as |x| is at most the largest from
// which the scale came.
__device__ inline std::uint32_t codes_of(float x0, float x1, float x2, float x3, float inv)
{
#pragma clang fp contract(off)
    constexpr float kWhole = 12582912.0f;
    const float p0 = x0 * inv, p1 = x1 * inv, p2 = x2 * inv, p3 = x3 * inv;
    const std::uint32_t a = __float_as_uint(p0 + kWhole), b = __float_as_uint(p1 + kWhole);
    const std::uint32_t c = __float_as_uint(p2 + kWhole), d = __float_as_uint(p3 + kWhole);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

// Old codes at a new scale.
__device__ inline std::uint32_t rescaled(std::uint32_t codes, float ratio)
{
    std::uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = quantise(static_cast<float>(static_cast<std::int8_t>(codes >> (8 * i))), ratio);
        out |= static_cast<std::uint32_t>(static_cast<std::uint8_t>(static_cast<std::int8_t>(q))) << (8 * i);
    }
    return out;
}

template <int kLane>
__device__ inline std::uint32_t from_quad(std::uint32_t x)  // lane kLane's of each four lanes
{
    return static_cast<std::uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), kLane * 0x55, 0xf, 0xf, true));
}

// One workgroup per (slot, kv head, keys or values), one wave per 16 tokens of
// the block: a lane holds token lane % 16's dims 16 (lane / 16) .. + 15 of
// every 64 in registers from the one read of the input to its codes.  That is
// the keys' layout already; values are transposed four tokens by four dims
// within four lanes.  Bound by memory: 27,600 tokens of 8 kv heads x 128 (170 MB
// in and out) take 57 us, 3.0 TB/s; 64 tokens 6.4 us, the way from the table
// through the scale to the row.
template <typename T, int CH>
__global__ __launch_bounds__(512) void k_kv_append(Append a)
{
    constexpr int P = CH * 64, kRow = P + 4;
    extern __shared__ std::uint8_t s_codes[];  // keys: [block tokens][kRow]
    __shared__ float s_top[8];
    __shared__ int s_bad[8];
    Write w;
    if (!find_write(a, blockIdx.x, &w)) {
        return;
    }
    const std::uint32_t head = blockIdx.y, which = blockIdx.z;
    const int lane = threadIdx.x % kWave, tile = threadIdx.x / kWave, waves = static_cast<int>(a.c.tokens) / 16;
    const int n = lane & 15, c = lane >> 4, D = static_cast<int>(a.c.dim);
    const bool begun = w.begin > 0;
    const std::size_t bh = static_cast<std::size_t>(w.id) * a.c.kv_heads + head;
    float* scales = which == 0 ? a.c.key_scale : a.c.value_scale;
    const float before = begun ? scales[bh] : 0.0f;
    const int token = tile * 16 + n;
    const bool fresh = token >= w.begin && token < w.end;
    const T* row = static_cast<const T*>(a.x[which]) + (w.row + (fresh ? token - w.begin : 0)) * a.token_stride[which] +
                   head * a.head_stride[which];

    float x[CH][16];
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        load_16<T>(row, i * 64 + c * 16, D, a.vector[which] != 0, x[i]);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            x[i][j] = fresh ? x[i][j] : 0.0f;
            bad |= !(fabsf(x[i][j]) < kInf);
            top = fmaxf(top, fabsf(x[i][j]));
        }
    }
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) top = fmaxf(top, __shfl_xor(top, k));
    const bool any_bad = __any(bad);
    if (lane == 0) {
        s_top[tile] = top;
        s_bad[tile] = any_bad;
    }
    __syncthreads();
    bad = any_bad;
    for (int i = 0; i < waves; ++i) {
        top = fmaxf(top, s_top[i]);
        bad |= s_bad[i] != 0;
    }
    float scale = top * kInv127;
    scale = bad || !(scale <= kScaleMax) ? __builtin_nanf("") : fmaxf(scale, kScaleMin);
    float ratio = 0.0f;
    if (begun) {
        scale = before != before || scale != scale ? __builtin_nanf("") : fmaxf(before, scale);
        ratio = before / scale;
    }
    const bool lost = scale != scale;  // no codes but zeros
    const float inv = lost ? 0.0f : 1.0f / scale;
    if (threadIdx.x == 0) {
        scales[bh] = scale;
        if (which == 0 && !begun) {
            a.c.weight[bh] = 0;
        }
    }

    std::int8_t* pool = (which == 0 ? a.c.keys : a.c.values) + bh * (static_cast<std::size_t>(a.c.tokens) * P) +
                        static_cast<std::size_t>(tile) * 16 * P;
    const bool keep = begun && ratio == 1.0f;  // old codes stay as they are
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        u32x4 q = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const std::uint32_t y = codes_of(x[i][4 * j], x[i][4 * j + 1], x[i][4 * j + 2], x[i][4 * j + 3], inv);
            q[j] = lost ? 0u : y;
        }
        if (which == 0) {
            u32x4* piece = reinterpret_cast<u32x4*>(pool + i * 1024) + lane;
            if (begun && !fresh && !keep) {
                const u32x4 old = *piece;
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = rescaled(old[j], ratio);
            }
            if (fresh || !keep) {
                *piece = q;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                *reinterpret_cast<std::uint32_t*>(s_codes + token * kRow + i * 64 + c * 16 + j * 4) = q[j];
            }
        } else {
            // lane r of four holds, for each j, byte r of the four lanes' words: the codes of
            // dim 16 c + 4 j + r of tokens 4 (n / 4) .. + 3
            const int r = n & 3, first = tile * 16 + (n & 12);
            const std::uint32_t pick = (static_cast<std::uint32_t>(r + 4) << 8) | static_cast<std::uint32_t>(r);
            std::uint32_t mask = 0;  // bytes of new tokens
#pragma unroll
            for (int k = 0; k < 4; ++k) mask |= first + k >= w.begin && first + k < w.end ? 0xffu << (8 * k) : 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const std::uint32_t lo = __builtin_amdgcn_perm(from_quad<1>(q[j]), from_quad<0>(q[j]), pick);
                const std::uint32_t hi = __builtin_amdgcn_perm(from_quad<3>(q[j]), from_quad<2>(q[j]), pick);
                std::uint32_t y = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
                std::uint32_t* at = reinterpret_cast<std::uint32_t*>(pool + i * 1024 + ((n >> 2) * 16 + 4 * j + r) * 16 + c * 4);
                if (mask == 0 && keep) {
                    continue;
                }
                if (begun && mask != 0xffffffffu) {
                    const std::uint32_t old = *at;
                    y = (y & mask) | ((keep ? old : rescaled(old, ratio)) & ~mask);
                }
                *at = y;
            }
        }
    }
    if (which != 0) {
        return;
    }
    __syncthreads();
    std::int8_t* bounds = a.c.bounds + bh * 2 * P;
    for (int d = threadIdx.x * 2; d < P; d += static_cast<int>(blockDim.x) * 2) {
        int lo[2] = {127, 127}, hi[2] = {-127, -127};
        if (begun) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                lo[u] = static_cast<int>(quantise(static_cast<float>(bounds[d + u]), ratio));
                hi[u] = static_cast<int>(quantise(static_cast<float>(bounds[P + d + u]), ratio));
            }
        }
#pragma unroll 4
        for (int k = w.begin; k < w.end; ++k) {
            const std::uint16_t two = *reinterpret_cast<const std::uint16_t*>(s_codes + k * kRow + d);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int q = static_cast<std::int8_t>(two >> (8 * u));
                lo[u] = q < lo[u] ? q : lo[u];
                hi[u] = q > hi[u] ? q : hi[u];
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            bounds[d + u] = static_cast<std::int8_t>(lo[u]);
            bounds[P + d + u] = static_cast<std::int8_t>(hi[u]);
        }
    }
}

// Blocks back as values: one wave per (entry, kv head, 16 tokens, keys or
// values).  Keys: a lane widens a token's 16 dims of every 64 and stores them
// as they are.  Values: four lanes transpose four tokens by four dims first,
// as append does.  The blocks of those 27,600 tokens (171 MB) take 37 us, 4.6 TB/s.
template <typename T>
__device__ inline void store_16(T* row, int d0, int dim, bool vector, std::uint32_t w0, std::uint32_t w1, std::uint32_t w2,
                                std::uint32_t w3, float scale)
{
    constexpr int kEach = 16 / sizeof(T);
    const std::uint32_t word[4] = {w0, w1, w2, w3};
    union {
        u32x4 v[sizeof(T)];
        T e[16];
    } u;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        u.e[i] = from_float<T>(static_cast<float>(static_cast<std::int8_t>(word[i / 4] >> (8 * (i % 4)))) * scale);
    }
    if (vector && dim % kEach == 0) {
#pragma unroll
        for (int i = 0; i < 16; i += kEach) {
            if (d0 + i < dim) *reinterpret_cast<u32x4*>(row + d0 + i) = u.v[i / kEach];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (d0 + i < dim) row[d0 + i] = u.e[i];
        }
    }
}

template <typename T, int CH>
__global__ __launch_bounds__(512) void k_kv_read(Cache c, const std::int32_t* ids, T* k_out, T* v_out, T* low, T* high,
                                                 std::uint32_t vector)
{
    constexpr int P = CH * 64;
    const std::uint32_t head = blockIdx.y, which = blockIdx.z;
    const std::int32_t id = ids[blockIdx.x];
    const bool inside = static_cast<std::uint32_t>(id) < c.blocks;
    const int D = static_cast<int>(c.dim), t = static_cast<int>(c.tokens);
    const int lane = threadIdx.x % kWave, tile = threadIdx.x / kWave, n = lane & 15, quarter = lane >> 4;
    const std::size_t bh = inside ? static_cast<std::size_t>(id) * c.kv_heads + head : 0;
    const std::size_t to = static_cast<std::size_t>(blockIdx.x) * c.kv_heads + head;
    const float scale = inside ? (which == 0 ? c.key_scale : c.value_scale)[bh] : 0.0f;
    const std::int8_t* pool = (which == 0 ? c.keys : c.values) + bh * (static_cast<std::size_t>(t) * P) +
                              static_cast<std::size_t>(tile) * 16 * P;
    T* row = (which == 0 ? k_out : v_out) + (to * t + tile * 16 + n) * D;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        std::uint32_t w[4];
        if (which == 0) {
            const u32x4 x = reinterpret_cast<const u32x4*>(pool + i * 1024)[lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = x[j];
        } else {
            const int r = n & 3;
            const std::uint32_t pick = (static_cast<std::uint32_t>(r + 4) << 8) | static_cast<std::uint32_t>(r);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const std::uint32_t x = *reinterpret_cast<const std::uint32_t*>(
                    pool + i * 1024 + ((n >> 2) * 16 + 4 * j + r) * 16 + quarter * 4);
                const std::uint32_t lo = __builtin_amdgcn_perm(from_quad<1>(x), from_quad<0>(x), pick);
                const std::uint32_t hi = __builtin_amdgcn_perm(from_quad<3>(x), from_quad<2>(x), pick);
                w[j] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = inside ? w[j] : 0u;
        store_16<T>(row, i * 64 + quarter * 16, D, vector != 0, w[0], w[1], w[2], w[3], scale);
    }
    if (which == 0) {
        for (int d = threadIdx.x; d < D; d += static_cast<int>(blockDim.x)) {
            const std::int8_t* b = c.bounds + bh * 2 * P + d;
            low[to * D + d] = from_float<T>(inside ? static_cast<float>(b[0]) * scale : 0.0f);
            high[to * D + d] = from_float<T>(inside ? static_cast<float>(b[P]) * scale : 0.0f);
        }
    }
}

// ---- select and evict -----------------------------------------------------

// The `want` largest of the n keys of a workgroup (want <= n; ties to the
// lower index): those above *threshold, and as many equal to it as the call
// returns.  All threads call it after a barrier behind the keys' stores.
// Digits of 8 bits from the highest bit in which two keys differ, a histogram
// of the keys that still match each, its suffix sums by one wave; it ends as
// soon as a digit's keys are all taken.
template <typename K, int kThreads>
__device__ std::uint32_t pick_threshold(const K* keys, std::uint32_t n, std::uint32_t want, K* threshold)
{
    __shared__ std::uint32_t bins[256];
    __shared__ K s_differ[kThreads / kWave];
    __shared__ std::uint32_t s_found[2];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    if (want == 0) {
        *threshold = ~K{0};
        return 0;
    }
    const K sample = keys[0];
    K differ = 0;
    for (std::uint32_t i = threadIdx.x; i < n; i += kThreads) differ |= keys[i] ^ sample;
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) differ |= __shfl_xor(differ, k);
    if (lane == 0) s_differ[wave] = differ;
    __syncthreads();
    differ = 0;
#pragma unroll
    for (int i = 0; i < kThreads / kWave; ++i) differ |= s_differ[i];
    int top = differ == 0 ? 0 : 64 - __clzll(static_cast<long long>(differ));  // bits in which keys differ
    K mask = top >= static_cast<int>(sizeof(K) * 8) ? K{0} : static_cast<K>(~K{0} << top);
    K prefix = sample & mask;
    std::uint32_t left = want;
    while (top > 0) {
        const int shift = top > 8 ? top - 8 : 0;
        const std::uint32_t digits = (1u << (top - shift)) - 1;
        for (int i = threadIdx.x; i < 256; i += kThreads) bins[i] = 0;
        __syncthreads();
        for (std::uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const K k = keys[i];
            if ((k & mask) == prefix) atomicAdd(&bins[static_cast<std::uint32_t>(k >> shift) & digits], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            std::uint32_t mine[4], sum = 0;  // lane 0 holds the highest digits
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                mine[i] = bins[255 - lane * 4 - i];
                sum += mine[i];
            }
            std::uint32_t upto = sum;
#pragma unroll
            for (int k = 1; k < kWave; k *= 2) {
                const std::uint32_t x = __shfl_up(upto, k);
                upto += lane >= k ? x : 0;
            }
            std::uint32_t above = upto - sum;
            if (above < left && upto >= left) {
                int i = 0;
                for (; i < 3 && above + mine[i] < left; ++i) above += mine[i];
                s_found[0] = 255 - lane * 4 - i;
                s_found[1] = left - above;
            }
        }
        __syncthreads();
        const std::uint32_t digit = s_found[0];
        left = s_found[1];
        prefix |= static_cast<K>(digit) << shift;
        mask |= static_cast<K>(digits) << shift;
        top = shift;
        if (bins[digit] == left) {  // every key of this digit is taken
            *threshold = prefix == 0 ? prefix : prefix - 1;
            return prefix == 0 ? left : 0;
        }
        __syncthreads();
    }
    *threshold = prefix;
    return left;
}

// Places in order of the n items of a workgroup that `above` or, for the
// first `equal` of them, `ties` names: calls put(i, place) for an item taken
// and skip(i, items taken before it) for one not.  Returns how many are taken.
template <int kThreads, typename A, typename P, typename S>
__device__ std::uint32_t place_in_order(std::uint32_t n, std::uint32_t equal, A about, P put, S skip)
{
    __shared__ unsigned long long s_wave[kThreads / kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const std::uint32_t each = (n + kThreads - 1) / kThreads;
    const std::uint32_t begin = threadIdx.x * each < n ? threadIdx.x * each : n;
    const std::uint32_t end = begin + each < n ? begin + each : n;
    unsigned long long mine = 0;  // above in the low half, ties in the high one
    for (std::uint32_t i = begin; i < end; ++i) {
        const int x = about(i);
        mine += x > 0 ? 1ull : x == 0 ? 1ull << 32 : 0ull;
    }
    unsigned long long upto = mine;
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) {
        const unsigned long long x = __shfl_up(upto, k);
        upto += lane >= k ? x : 0ull;
    }
    if (lane == kWave - 1) s_wave[wave] = upto;
    __syncthreads();
    unsigned long long before = upto - mine, all = 0;
#pragma unroll
    for (int i = 0; i < kThreads / kWave; ++i) {
        before += i < wave ? s_wave[i] : 0ull;
        all += s_wave[i];
    }
    std::uint32_t over = static_cast<std::uint32_t>(before), tied = static_cast<std::uint32_t>(before >> 32);
    for (std::uint32_t i = begin; i < end; ++i) {
        const int x = about(i);
        const std::uint32_t place = over + (tied < equal ? tied : equal);
        if (x > 0 || (x == 0 && tied < equal)) {
            put(i, place);
        } else {
            skip(i, place);
        }
        over += x > 0;
        tied += x == 0;
    }
    const std::uint32_t ties = static_cast<std::uint32_t>(all >> 32);
    return static_cast<std::uint32_t>(all) + (ties < equal ? ties : equal);
}

struct Select {
    Cache c;
    Batch b;
    const void* q;
    std::int64_t q_token, q_head;
    std::uint32_t group, count, keep_first, keep_last;
    std::uint32_t per, share; // tokens per group of the scoring pass, blocks per workgroup
    std::uint32_t staged;     // the choice reads its keys from LDS
    std::uint32_t* keys;      // [tokens, kv heads, width]
    std::int32_t* selected;   // [tokens, kv heads, count]
};

__device__ inline std::uint32_t ordered(float x)
{
    const std::uint32_t u = __float_as_uint(x);
    return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}

// Blocks that a token that sees `seen` tokens sees.
__device__ inline std::uint32_t select_blocks(const Select& a, std::int64_t seen)
{
    const std::int64_t nb = seen <= 0 ? 0 : (seen + a.c.tokens - 1) / a.c.tokens;
    return nb < static_cast<std::int64_t>(a.b.width) ? static_cast<std::uint32_t>(nb) : a.b.width;
}

// The group's queries of a token as codes of one scale, summed over the heads
// by sign (what meets the low bounds, then what meets the high ones), each sum
// as 128 * [0] + [1] of two signed bytes.  One wave; [2][2 * dims] bytes.
template <typename T>
__device__ void query_codes(const Select& a, std::int64_t row, std::uint32_t head, int lane, std::int8_t* to)
{
    const int P = static_cast<int>(a.c.dims), D = static_cast<int>(a.c.dim), G = static_cast<int>(a.group);
    const T* q = static_cast<const T*>(a.q) + row * a.q_token + static_cast<std::int64_t>(head) * G * a.q_head;
    float top = 0.0f;
    for (int g = 0; g < G; ++g) {
        for (int d = lane; d < D; d += kWave) top = fmaxf(top, fabsf(to_float(q[g * a.q_head + d])));
    }
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) top = fmaxf(top, __shfl_xor(top, k));
    const float inv = 1.0f / fmaxf(top * kInv127, kQueryScaleMin);
    for (int d = lane; d < P; d += kWave) {
        std::int32_t sum[2] = {0, 0};
        for (int g = 0; g < G && d < D; ++g) {
            const std::int32_t code = static_cast<std::int32_t>(quantise(to_float(q[g * a.q_head + d]), inv));
            sum[code > 0] += code;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const std::int32_t hi = (sum[i] + 64) >> 7;
            to[i * P + d] = static_cast<std::int8_t>(hi);
            to[2 * P + i * P + d] = static_cast<std::int8_t>(sum[i] - hi * 128);
        }
    }
}

// Scores of a wave's 32 blocks for up to 8 query tokens, 16 at a time: bounds are the
// matrix units' second operand (a lane's block is lane % 16), the tokens'
// codes the first (rows 2 t and 2 t + 1 are token t's two bytes), so that a
// lane ends with its block's scores of tokens 2 (lane / 16) and the next.
template <int CH>
__device__ inline void block_scores(const Cache& c, const std::int32_t (&id)[2], std::uint32_t head, int quarter,
                                    const i32x4 (&codes)[CH * 2], float (&score)[2][2])
{
    i32x4 x[2][CH * 2];
    float scale[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const std::size_t bh = static_cast<std::size_t>(id[u] < 0 ? 0 : id[u]) * c.kv_heads + head;
        const i32x4* bounds = reinterpret_cast<const i32x4*>(c.bounds + bh * (CH * 128));
#pragma unroll
        for (int i = 0; i < CH * 2; ++i) x[u][i] = bounds[i * 4 + quarter];
        scale[u] = c.key_scale[bh];
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        i32x4 s = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < CH * 2; ++i) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(codes[i], x[u][i], s, 0, 0, 0);
        score[u][0] = static_cast<float>(s[0] * 128 + s[1]) * scale[u];
        score[u][1] = static_cast<float>(s[2] * 128 + s[3]) * scale[u];
    }
}

template <int CH>
__device__ inline void load_codes(const std::int8_t* from, int token, int part, int quarter, i32x4 (&codes)[CH * 2])
{
    const i32x4* p = reinterpret_cast<const i32x4*>(from + (token * 2 + part) * (CH * 128));
#pragma unroll
    for (int i = 0; i < CH * 2; ++i) codes[i] = p[i * 4 + quarter];
}

// A block's key: 0 for one that is not there, and above every score's for a
// scale that is not a number.
__device__ inline std::uint32_t score_key(std::int32_t id, float score)
{
    return id < 0 ? 0u : ordered(score != score ? kInf : score);
}

// Writes a row's choice of its nb keys: the first and last that are always
// in, the best of the others.
template <int kThreads>
__device__ void write_choice(const Select& a, const std::uint32_t* keys, std::uint32_t nb, std::int32_t* out)
{
    std::uint32_t threshold = 0, equal = 0, lo = 0, hi = 0;  // lo..hi: those that compete
    if (nb > a.count) {
        lo = a.keep_first;
        hi = nb - a.keep_last;
        std::uint32_t sure = 0;  // of those always in, the ones that are there
        const std::uint32_t always = a.keep_first + a.keep_last;
        for (std::uint32_t base = 0; base < always; base += kThreads) {
            const std::uint32_t i = base + threadIdx.x;
            sure += __syncthreads_count(i < always && keys[i < lo ? i : hi + i - lo] != 0);
        }
        const std::uint32_t want = a.count - sure < hi - lo ? a.count - sure : hi - lo;
        equal = pick_threshold<std::uint32_t, kThreads>(keys + lo, hi - lo, want, &threshold);
    }
    // keys of 0, blocks that are not there, are never taken
    const auto about = [&](std::uint32_t i) {
        const std::uint32_t k = keys[i];
        if (k == 0) return -1;
        return i < lo || i >= hi || k > threshold ? 1 : k == threshold ? 0 : -1;
    };
    const std::uint32_t done = place_in_order<kThreads>(
        nb, equal, about, [&](std::uint32_t i, std::uint32_t at) { out[at] = static_cast<std::int32_t>(i); },
        [](std::uint32_t, std::uint32_t) {});
    for (std::uint32_t i = done + threadIdx.x; i < a.count; i += kThreads) out[i] = -1;
}

// Scores and choice of one query token and kv head in one workgroup, the keys
// in LDS.  64 sequences of 1024..32768 tokens (155 MB of bounds) take 66 us, 24
// of them without the bounds and 60 without the choice; 64 of equal length 23.5
// us at 8192 tokens, 45.7 at 16384 and 80.3 at 32768, so that once running the
// bounds of a block and head, 256 bytes at random places, come at 3.9 TB/s
// (about 5 with the cache lines of their scales), and the longest rows end last.
template <typename T, int CH>
__global__ __launch_bounds__(kPickThreads) void k_kv_select(Select a)
{
    extern __shared__ std::uint32_t s_keys[];
    __shared__ i32x4 s_codes[CH * 16];
    const std::uint32_t token = blockIdx.x / a.c.kv_heads, head = blockIdx.x % a.c.kv_heads;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    Group g;
    std::uint32_t nb = 0;
    if (find_group(a.b, token, 1, &g)) nb = select_blocks(a, g.seen);
    std::int8_t* codes_at = reinterpret_cast<std::int8_t*>(s_codes);
    if (wave == 0 && nb > a.count) query_codes<T>(a, token, head, lane, codes_at);
    __syncthreads();
    const int quarter = lane >> 4;
    i32x4 codes[CH * 2];
    // rows past the token's two are not looked at: they repeat them
    load_codes<CH>(codes_at, 0, lane & 1, quarter, codes);
    const auto look_up = [&](std::uint32_t at, std::int32_t (&id)[2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const std::uint32_t blk = at + u * 16 + (lane & 15);
            id[u] = blk < nb ? block_at(a.c, a.b, g.seq, blk) : -1;
        }
    };
    std::int32_t next[2];
    look_up(wave * 32, next);
    for (std::uint32_t at = wave * 32; at < nb; at += kPickThreads / kWave * 32) {
        const std::int32_t id[2] = {next[0], next[1]};
        look_up(at + kPickThreads / kWave * 32, next);
        std::uint32_t key[2] = {id[0] < 0 ? 0u : 1u, id[1] < 0 ? 0u : 1u};
        if (nb > a.count) {
            float score[2][2];
            block_scores<CH>(a.c, id, head, quarter, codes, score);
            key[0] = score_key(id[0], score[0][0]);
            key[1] = score_key(id[1], score[1][0]);
        }
        // quarter u stores tile u's keys
        const std::uint32_t blk = at + (lane & 31);
        if (blk < nb && lane < 32) s_keys[blk] = quarter == 0 ? key[0] : key[1];
    }
    __syncthreads();
    write_choice<kPickThreads>(a, s_keys, nb, a.selected + static_cast<std::size_t>(blockIdx.x) * a.count);
}

// Scores of groups of up to 8 tokens of a sequence, to global memory.  1,001
// tokens of 4 kv heads over 1,001 blocks: 26 us, the codes' preparation and
// the way through the table more than the bounds; their choice 21 us.
template <typename T, int CH>
__global__ __launch_bounds__(256) void k_kv_score(Select a)
{
    __shared__ i32x4 s_codes[8 * CH * 16];
    const std::uint32_t slot = blockIdx.x / a.c.kv_heads, head = blockIdx.x % a.c.kv_heads;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, quarter = lane >> 4;
    Group g;
    if (!find_group(a.b, slot, a.per, &g)) {
        return;
    }
    const std::uint32_t nb = select_blocks(a, g.seen + g.count - 1);
    if (blockIdx.y * a.share >= nb) {
        return;
    }
    std::int8_t* codes_at = reinterpret_cast<std::int8_t*>(s_codes);
    for (int t = wave; t < g.count; t += 4) query_codes<T>(a, g.row + t, head, lane, codes_at + t * (CH * 256));
    __syncthreads();
    i32x4 codes[CH * 2];
    const int t = (lane & 15) / 2 < g.count ? (lane & 15) / 2 : 0;
    load_codes<CH>(codes_at, t, lane & 1, quarter, codes);
    const std::uint32_t end = (blockIdx.y + 1) * a.share < nb ? (blockIdx.y + 1) * a.share : nb;
    const auto look_up = [&](std::uint32_t at, std::int32_t (&id)[2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const std::uint32_t blk = at + u * 16 + (lane & 15);
            id[u] = blk < end ? block_at(a.c, a.b, g.seq, blk) : -1;
        }
    };
    std::int32_t next[2];
    look_up(blockIdx.y * a.share + wave * 32, next);
    for (std::uint32_t at = blockIdx.y * a.share + wave * 32; at < end; at += 128) {
        const std::int32_t id[2] = {next[0], next[1]};
        look_up(at + 128, next);
        float score[2][2];
        block_scores<CH>(a.c, id, head, quarter, codes, score);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const std::uint32_t blk = at + u * 16 + (lane & 15);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int token = quarter * 2 + i;
                if (token < g.count && blk < end) {
                    a.keys[(static_cast<std::size_t>(g.row + token) * a.c.kv_heads + head) * a.b.width + blk] =
                        score_key(id[u], score[u][i]);
                }
            }
        }
    }
}

// The choice of each row of those keys.
__global__ __launch_bounds__(256) void k_kv_pick(Select a)
{
    extern __shared__ std::uint32_t s_keys[];
    const std::uint32_t token = blockIdx.x / a.c.kv_heads;
    std::uint32_t slot = token;
    if (a.b.first != nullptr) {
        // slot_base with one token per slot
        slot = token + last_not_above(a.b.seqs, token, [&](std::uint32_t i) { return static_cast<std::uint32_t>(a.b.first[i]); });
    }
    Group g;
    const std::uint32_t nb = a.b.seqs != 0 && find_group(a.b, slot, 1, &g) ? select_blocks(a, g.seen) : 0;
    const std::uint32_t* keys = a.keys + static_cast<std::size_t>(blockIdx.x) * a.b.width;
    if (a.staged != 0) {
        for (std::uint32_t i = threadIdx.x; i < nb; i += 256) s_keys[i] = keys[i];
        __syncthreads();
        keys = s_keys;
    }
    write_choice<256>(a, keys, nb, a.selected + static_cast<std::size_t>(blockIdx.x) * a.count);
}

struct Evict {
    const unsigned long long* weight;
    std::uint32_t blocks, kv_heads, tokens;
    const std::int32_t* table;
    const std::int32_t* lens;
    std::uint32_t seqs, width, stride, keep, keep_first, keep_last;
    unsigned long long* keys;  // [seqs, width]
    std::int32_t* out_table;   // [seqs, width]
    std::int32_t* out_lens;
    std::int32_t* freed;       // [seqs, width]
    std::int32_t* freed_count;
};

// One workgroup per sequence, the keys in LDS if they fit (kStaged).  A
// block's key is its summed weight plus 1; a table entry that names no block
// has key 0 and goes first.  Latency bounds it: 6.6 us for 3 sequences of up to
// 313 blocks, 13.6 for 64 of up to 2,048 (5.3 MB), of which each digit's
// histogram and scan is about 1.5.
template <bool kStaged>
__global__ __launch_bounds__(kPickThreads) void k_kv_evict(Evict a)
{
    extern __shared__ unsigned long long s_weights[];
    const std::uint32_t s = blockIdx.x;
    const std::int64_t len = a.lens[s];
    const std::int64_t nb64 = len <= 0 ? 0 : (len + a.tokens - 1) / a.tokens;
    const std::uint32_t nb = nb64 < static_cast<std::int64_t>(a.width) ? static_cast<std::uint32_t>(nb64) : a.width;
    const std::int32_t* table = a.table + static_cast<std::size_t>(s) * a.stride;
    unsigned long long* keys = kStaged ? s_weights : a.keys + static_cast<std::size_t>(s) * a.width;
    unsigned long long threshold = 0;
    std::uint32_t equal = 0, lo = 0, hi = 0;
    if (nb > a.keep) {
        lo = a.keep_first;
        hi = nb - a.keep_last;
        for (std::uint32_t i = threadIdx.x; i < nb; i += kPickThreads) {
            const std::uint32_t id = static_cast<std::uint32_t>(table[i]);
            unsigned long long key = 0;
            if (id < a.blocks) {
                const unsigned long long* w = a.weight + static_cast<std::size_t>(id) * a.kv_heads;
                key = 1;
#pragma unroll 8
                for (std::uint32_t h = 0; h < a.kv_heads; ++h) key += w[h];
            }
            keys[i] = key;
        }
        __syncthreads();
        equal = pick_threshold<unsigned long long, kPickThreads>(keys + lo, hi - lo, a.keep - a.keep_first - a.keep_last, &threshold);
    }
    std::int32_t* kept = a.out_table + static_cast<std::size_t>(s) * a.width;
    std::int32_t* freed = a.freed + static_cast<std::size_t>(s) * a.width;
    const auto about = [&](std::uint32_t i) {
        if (i < lo || i >= hi) return 1;
        const unsigned long long k = keys[i];
        return k > threshold ? 1 : k == threshold ? 0 : -1;
    };
    const std::uint32_t done = place_in_order<kPickThreads>(
        nb, equal, about, [&](std::uint32_t i, std::uint32_t at) { kept[at] = table[i]; },
        [&](std::uint32_t i, std::uint32_t before) { freed[i - before] = table[i]; });
    for (std::uint32_t i = done + threadIdx.x; i < a.width; i += kPickThreads) kept[i] = -1;
    for (std::uint32_t i = nb - done + threadIdx.x; i < a.width; i += kPickThreads) freed[i] = -1;
    if (threadIdx.x == 0) {
        a.out_lens[s] = static_cast<std::int32_t>(len - static_cast<std::int64_t>(nb - done) * a.tokens);
        a.freed_count[s] = static_cast<std::int32_t>(nb - done);
    }
}

// ---- host -----------------------------------------------------------------

// A launch dimension holds fewer than 2^32 threads, a workgroup at most 1024.
constexpr std::size_t kMostGroups = (std::size_t{1} << 22) - 1;

bool aligned16(const void* p) { return (reinterpret_cast<std::uintptr_t>(p) & 15u) == 0; }

int checked(hipError_t e) { return e == hipSuccess ? HBFSIM_OK : HBFSIM_CUDA_ERROR; }

// The cache's own fields; pools may be asked for or not.
int take_cache(const hbfsim_amd_kv_cache* in, Cache* out)
{
    if (in == nullptr || in->struct_size != sizeof(*in)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    const bool tokens_ok = in->block_tokens == 16 || in->block_tokens == 32 ||
                           in->block_tokens == 64 || in->block_tokens == 128;
    if (in->blocks == 0 || in->blocks > 0x7fffffffu || in->kv_heads == 0 || in->kv_heads > 1024 ||
        in->head_dim == 0 || in->head_dim > 256 || !tokens_ok) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (in->d_keys == nullptr || in->d_values == nullptr || in->d_key_scale == nullptr ||
        in->d_value_scale == nullptr || in->d_bounds == nullptr || in->d_weight == nullptr ||
        !aligned16(in->d_keys) || !aligned16(in->d_values) || !aligned16(in->d_bounds)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    out->keys = in->d_keys;
    out->values = in->d_values;
    out->key_scale = in->d_key_scale;
    out->value_scale = in->d_value_scale;
    out->bounds = in->d_bounds;
    out->weight = reinterpret_cast<unsigned long long*>(in->d_weight);
    out->blocks = in->blocks;
    out->kv_heads = in->kv_heads;
    out->dim = in->head_dim;
    out->dims = (in->head_dim + 63) / 64 * 64;
    out->tokens = in->block_tokens;
    out->tile_shift = in->block_tokens == 16 ? 0 : in->block_tokens == 32 ? 1 : in->block_tokens == 64 ? 2 : 3;
    return HBFSIM_OK;
}

int take_batch(const hbfsim_amd_kv_batch* in, const Cache& c, Batch* out)
{
    if (in == nullptr || in->struct_size != sizeof(*in) || in->table_stride < in->table_width) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    // positions are 32-bit signed, with room for a tile beyond the last
    if (static_cast<std::uint64_t>(in->table_width) * c.tokens > 0x7fffff00u ||
        in->tokens > 0x7fffff00u || in->seqs > 0x7fffff00u) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (in->d_first == nullptr && in->tokens != in->seqs) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (in->seqs != 0 && in->tokens != 0 && (in->d_lens == nullptr || (in->table_width != 0 && in->d_table == nullptr))) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    out->table = in->d_table;
    out->lens = in->d_lens;
    out->first = in->d_first;
    out->seqs = in->seqs;
    out->width = in->table_width;
    out->stride = in->table_stride;
    out->tokens = in->tokens;
    return HBFSIM_OK;
}

bool two_byte(std::uint32_t type) { return type == HBFSIM_AMD_KV_BF16 || type == HBFSIM_AMD_KV_F16; }

// How attend cuts its work: from the call's host-side sizes alone.
struct Cut {
    std::uint32_t many;  // row tiles per wave of the many-row form, or 0
    std::uint32_t per, row_tiles, rows, units, split, splits;
    std::size_t partial, stats, lse, tile_sums, bytes;
};

std::size_t up256(std::size_t x) { return (x + 255) & ~std::size_t{255}; }

// Row tiles per wave that fit the registers of two waves per SIMD (16 chunks
// of 2048 tokens over 16384, D = 64: 5.84 / 5.14 / 5.38 ms with 3 / 4 / 5, D =
// 128: 9.06 / 8.53 / 14.2 with 2 / 3 / 4; 8 of 1024 over 8192, D = 192: 2.22 /
// 1.95 / 6.92 with 1 / 2 / 3, D = 256: 3.59 / 3.95 with 1 / 2: more spill).
std::uint32_t many_tiles(std::uint32_t dims) { return 5 - dims / 64; }

Cut cut_few(const Cache& c, const Batch& b, std::uint32_t heads, std::uint32_t count)
{
    Cut k{};
    const std::uint32_t group = heads / c.kv_heads;
    k.per = b.first == nullptr || count != 0 || group > 8 ? 1 : 16 / group;
    k.row_tiles = group > 16 ? (group + 15) / 16 : 1;
    k.rows = k.per * group < 16 ? k.per * group : 16;
    k.units = b.first == nullptr ? b.seqs : b.tokens / k.per + b.seqs;
    const std::uint64_t longest = static_cast<std::uint64_t>(count != 0 ? count : b.width) * c.tokens;
    const std::uint64_t pairs = static_cast<std::uint64_t>(k.units) * c.kv_heads * k.row_tiles;
    // Splits of 2048 tokens (64 sequences of 1024..32768 tokens: 422 us and 7 of
    // merge, with 1024 442 + 8, with 4096 427 + 5), shorter where they would not
    // fill the card.  Up to 1024 tokens take one and no second launch: one
    // sequence of 1024 takes 12.1 us in one split, 7.7 + 3.1 and a launch in
    // four; of 1536, 15.3 against 7.7 + 3.4.
    std::uint64_t split = 2048;
    while (longest > 1024 && split > 256 && pairs * ((longest + split - 1) / split) < 1024) split /= 2;
    k.split = static_cast<std::uint32_t>(split);
    k.splits = longest == 0 ? 1 : static_cast<std::uint32_t>((longest + split - 1) / split);
    return k;
}

Cut cut_many(const Cache& c, const Batch& b, std::uint32_t heads)
{
    Cut k{};
    const std::uint32_t group = heads / c.kv_heads;
    k.many = many_tiles(c.dims);
    const std::uint32_t room = 4 * k.many * 16;
    k.per = room / group;
    k.row_tiles = 1;
    k.rows = k.per * group;
    k.units = b.tokens / k.per + b.seqs;
    const std::uint64_t longest = static_cast<std::uint64_t>(b.width) * c.tokens;
    const std::uint64_t groups = static_cast<std::uint64_t>(k.units) * c.kv_heads;
    // Two workgroups fit a CU; splits fill the last round of them, each at
    // the price of its partial sums' round trip.  Chunks of 2,048 tokens over
    // 16,384 (8 kv heads, D = 128) take, with 1 / 2 / 3 / 4 splits and their
    // merge, 839 / 730 / 719 / 704 us for one of them (0.7 rounds), 1,285 /
    // 1,245 / 1,264 / 1,253 for two, 1,917 / 1,746 / 1,721 / 1,759 for three,
    // 3,383 / 3,537 / 3,564 / 3,565 for six (4.1), 4,128 / 4,291 / 4,376 / 4,476
    // for eight.  The table's width stands for the lengths, which the host does
    // not know: a table much wider than they are gives splits without work.
    std::uint64_t best = 1;
    double score = 0.0;
    for (std::uint64_t s = 1; s <= 16 && (s == 1 || (groups < 2048 && longest / s >= 256)); ++s) {
        const double rounds = static_cast<double>(groups * s) / 512.0;
        const double whole = static_cast<double>(static_cast<std::uint64_t>((groups * s + 511) / 512));
        const double got = rounds / whole / (s == 1 ? 1.0 : 1.0 + 0.03 * static_cast<double>(s));
        if (got > score * 1.02) {
            score = got;
            best = s;
        }
    }
    const std::uint64_t split = longest == 0 ? 64 : ((longest + best - 1) / best + 63) / 64 * 64;
    k.split = static_cast<std::uint32_t>(split);
    k.splits = longest == 0 ? 1 : static_cast<std::uint32_t>((longest + split - 1) / split);
    return k;
}

Cut cut_attend(const Cache& c, const Batch& b, std::uint32_t heads, std::uint32_t count, bool accumulate)
{
    const std::uint32_t group = heads / c.kv_heads;
    // The many-row form once a sequence's share of the step comes near a
    // workgroup's rows: 16 sequences of 8192 tokens (4 heads a kv head, D = 128)
    // take, merge and all, 142 us in the few-row form and 180 in this with 24
    // tokens (96 of 192 rows), 179 and 171 with 32, 268 and 244 with 48, 514 and
    // 322 with 96.  One sequence of 4096 tokens, which fills the card with
    // neither: 84 and 67 with 400 tokens, but 30 and 44 with 48.
    const std::uint64_t room = 4 * many_tiles(c.dims) * 16;
    const bool many = b.first != nullptr && count == 0 && group <= room &&
                      static_cast<std::uint64_t>(b.tokens) * group * 5 >= room * b.seqs * 4;
    Cut k = many ? cut_many(c, b, heads) : cut_few(c, b, heads, count);
    if (k.splits > 1) {
        const std::size_t cells = static_cast<std::size_t>(k.units) * c.kv_heads * k.row_tiles * k.splits * k.rows;
        k.stats = up256(cells * c.dims * sizeof(float));
        k.lse = k.stats + up256(cells * 2 * sizeof(float));
    }
    k.tile_sums = k.lse + (accumulate ? up256(static_cast<std::size_t>(b.tokens) * heads * sizeof(float)) : 0);
    k.bytes = k.tile_sums;
    if (accumulate && k.many == 0) {
        k.bytes += up256(static_cast<std::size_t>(k.units) * c.kv_heads * k.row_tiles * b.width * (c.tokens / 16) * k.rows * sizeof(float));
    }
    return k;
}

// Whether the output [tokens][heads][dim] at `out` shares memory with the
// query rows; `same` if it is they, row for row.  Two-byte elements.
bool overlaps(std::uintptr_t q, std::int64_t token_stride, std::int64_t head_stride, std::uintptr_t out, std::uint32_t tokens,
              std::uint32_t heads, std::uint32_t dim, bool* same)
{
    const std::int64_t row = std::int64_t{2} * dim, whole = row * heads * tokens;
    const std::int64_t t = 2 * token_stride, h = 2 * head_stride, last_t = (tokens - 1) * t, last_h = (heads - 1) * h;
    *same = q == out && (tokens == 1 || t == row * heads) && (heads == 1 || h == row);
    // distances from the output's first byte
    const std::int64_t at = static_cast<std::int64_t>(q - out);
    const std::int64_t lo = at + (last_t < 0 ? last_t : 0) + (last_h < 0 ? last_h : 0);
    const std::int64_t hi = at + (last_t > 0 ? last_t : 0) + (last_h > 0 ? last_h : 0) + row;
    if (lo >= whole || hi <= 0) {
        return false;
    }
    // within the rows' span: between them, perhaps
    for (std::uint32_t i = 0; i < tokens; ++i) {
        for (std::uint32_t j = 0; j < heads; ++j) {
            const std::int64_t x = at + i * t + j * h;
            if (x < whole && x + row > 0) {
                return true;
            }
        }
    }
    return false;
}

template <typename T, int CH>
void launch_append(const Append& a, std::uint32_t slots, hipStream_t stream)
{
    const std::size_t lds = static_cast<std::size_t>(a.c.tokens) * (CH * 64 + 4);
    hipLaunchKernelGGL((k_kv_append<T, CH>), dim3(slots, a.c.kv_heads, 2), dim3(a.c.tokens * 4), lds, stream, a);
}

template <typename T>
void run_append(const Append& a, std::uint32_t slots, hipStream_t stream)
{
    switch (a.c.dims / 64) {
    case 1: launch_append<T, 1>(a, slots, stream); break;
    case 2: launch_append<T, 2>(a, slots, stream); break;
    case 3: launch_append<T, 3>(a, slots, stream); break;
    default: launch_append<T, 4>(a, slots, stream); break;
    }
}

template <typename T, int CH>
void launch_read(const Cache& c, const std::int32_t* ids, std::uint32_t n, void* k, void* v, void* low, void* high,
                 std::uint32_t vector, hipStream_t stream)
{
    hipLaunchKernelGGL((k_kv_read<T, CH>), dim3(n, c.kv_heads, 2), dim3(c.tokens * 4), 0, stream, c, ids, static_cast<T*>(k),
                       static_cast<T*>(v), static_cast<T*>(low), static_cast<T*>(high), vector);
}

template <typename T>
void run_read(const Cache& c, const std::int32_t* ids, std::uint32_t n, void* k, void* v, void* low, void* high,
              std::uint32_t vector, hipStream_t stream)
{
    switch (c.dims / 64) {
    case 1: launch_read<T, 1>(c, ids, n, k, v, low, high, vector, stream); break;
    case 2: launch_read<T, 2>(c, ids, n, k, v, low, high, vector, stream); break;
    case 3: launch_read<T, 3>(c, ids, n, k, v, low, high, vector, stream); break;
    default: launch_read<T, 4>(c, ids, n, k, v, low, high, vector, stream); break;
    }
}

// Keys of a row that a choosing workgroup holds in LDS.
constexpr std::size_t kMostStaged = std::size_t{128} << 10;

// A kernel asks for more LDS than the 64 KiB that it has unasked, its own
// arrays among them.
bool lds_allowed(const void* kernel, std::size_t bytes)
{
    return bytes <= (std::size_t{48} << 10) ||
           hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) == hipSuccess;
}

// One workgroup per row does it all where there are rows enough to fill the
// card and no other token reads the same bounds: 64 sequences of 16384..32768
// tokens and 8 kv heads take 72 us in one launch and 63 + 12 in two, 32 take
// 43 and 34 + 12, 16 take 29 and 17 + 11, 8 take 29 and 13 + 10.
bool select_in_one(const Cache& c, const Batch& b)
{
    return b.first == nullptr && static_cast<std::uint64_t>(b.tokens) * c.kv_heads >= 128 &&
           static_cast<std::size_t>(b.width) * sizeof(std::uint32_t) <= kMostStaged;
}

std::size_t select_bytes(const Cache& c, const Batch& b)
{
    return select_in_one(c, b) ? 0
                               : static_cast<std::size_t>(b.tokens) * c.kv_heads * b.width * sizeof(std::uint32_t);
}

// Groups of up to 8 tokens of the scoring launch.
std::uint32_t score_slots(const Batch& b) { return b.first == nullptr ? b.seqs : b.tokens / 8 + b.seqs; }

template <typename T, int CH>
bool launch_select(Select& a, bool one, hipStream_t stream)
{
    const std::size_t keys = static_cast<std::size_t>(a.b.width) * sizeof(std::uint32_t);
    const std::uint32_t rows = a.b.tokens * a.c.kv_heads;
    if (one) {
        if (!lds_allowed(reinterpret_cast<const void*>(&k_kv_select<T, CH>), keys)) {
            return false;
        }
        hipLaunchKernelGGL((k_kv_select<T, CH>), dim3(rows), dim3(kPickThreads), keys, stream, a);
        return true;
    }
    if (a.b.width != 0 && a.b.seqs != 0) {
        a.per = a.b.first == nullptr ? 1 : 8;
        const std::uint32_t slots = score_slots(a.b);
        a.share = 256;
        while (a.share < 4096 && static_cast<std::uint64_t>(slots) * a.c.kv_heads * (a.b.width / a.share) > 4096) a.share *= 2;
        while (a.b.width / a.share > 65534) a.share *= 2;
        hipLaunchKernelGGL((k_kv_score<T, CH>), dim3(slots * a.c.kv_heads, (a.b.width + a.share - 1) / a.share), dim3(256), 0,
                           stream, a);
    }
    a.staged = keys <= kMostStaged ? 1 : 0;
    if (a.staged != 0 && !lds_allowed(reinterpret_cast<const void*>(&k_kv_pick), keys)) {
        return false;
    }
    hipLaunchKernelGGL(k_kv_pick, dim3(rows), dim3(256), a.staged != 0 ? keys : 0, stream, a);
    return true;
}

template <typename T>
bool run_select(Select& a, bool one, hipStream_t stream)
{
    switch (a.c.dims / 64) {
    case 1: return launch_select<T, 1>(a, one, stream);
    case 2: return launch_select<T, 2>(a, one, stream);
    case 3: return launch_select<T, 3>(a, one, stream);
    default: return launch_select<T, 4>(a, one, stream);
    }
}

template <typename T, int CH>
bool launch_attend(Attend a, const Cut& k, bool accumulate, hipStream_t stream)
{
    constexpr int RT = 5 - CH;
    const std::uint32_t groups = k.units * a.pairs;
    const std::uint32_t clearing = a.b.first == nullptr ? 0 : a.b.tokens < 128 ? a.b.tokens : 128;
    if (a.b.seqs == 0) {
        hipLaunchKernelGGL((k_kv_clear_rest<T>), dim3(clearing), dim3(256), 0, stream, a);
        return true;
    }
    a.groups = groups;
    if (k.many != 0) {
        const std::size_t lds = (CH <= 2 ? 32 : 16) * 1024 * CH;
        if (!lds_allowed(reinterpret_cast<const void*>(&k_kv_attend_many<T, CH, RT>), lds)) {
            return false;
        }
        hipLaunchKernelGGL((k_kv_attend_many<T, CH, RT>), dim3(groups, k.splits), dim3(256), lds, stream, a);
    } else {
        const std::size_t lds = 4 * k.rows * (CH * 64 + 4) * sizeof(float);
        // Codes pass the caches where a workgroup is alone with them: not where several units
        // of a sequence read the same blocks, of a selection either.  Marked / cached: 2 chunks of
        // 1,001 tokens (8 kv heads, D = 128) over 64 / 128 / 256 selected blocks 510 / 360, 895 / 645
        // and 1,545 / 1,170 us; 32 sequences of 4 tokens 49 / 51, 90 / 87 and 171 / 145.
        const bool once = k.row_tiles == 1 && (a.b.first == nullptr || a.b.tokens <= k.per * a.b.seqs);
        void (*kernel)(Attend) = accumulate ? once ? k_kv_attend<T, CH, 4, true, true> : k_kv_attend<T, CH, 4, true, false>
                                 : once     ? k_kv_attend<T, CH, 4, false, true>
                                            : k_kv_attend<T, CH, 4, false, false>;
        if (!lds_allowed(reinterpret_cast<const void*>(kernel), lds)) {
            return false;
        }
        hipLaunchKernelGGL(kernel, dim3(groups, k.splits), dim3(256), lds, stream, a);
    }
    // 24 sequences of 12 / 16 / 32 splits: 5.5 / 5.6 / 6.3 us by rows, 5.4 / 6.4 / 10.1 by quads of dims
    if (k.splits > 12) {
        hipLaunchKernelGGL((k_kv_merge<T>), dim3(groups + clearing, k.rows), dim3(256), 0, stream, a);
    } else if (k.splits > 1) {
        const std::uint32_t at_once = 1024 / a.c.dims;
        hipLaunchKernelGGL((k_kv_merge_few<T>), dim3(groups + clearing, (k.rows + at_once - 1) / at_once), dim3(256), 0, stream, a);
    } else if (clearing != 0) {
        hipLaunchKernelGGL((k_kv_clear_rest<T>), dim3(clearing), dim3(256), 0, stream, a);
    }
    if (!accumulate || a.b.width == 0) {
    } else if (k.many == 0) {
        hipLaunchKernelGGL(k_kv_weigh, dim3(groups, (a.b.width + 255) / 256), dim3(256), 0, stream, a);
    } else {
        const Cut few = cut_few(a.c, a.b, a.heads, 0);
        a.per = few.per;
        a.row_tiles = few.row_tiles;
        a.pairs = a.c.kv_heads * few.row_tiles;
        const std::uint32_t z = a.b.width / 64 < 65535 ? (a.b.width + 63) / 64 : 65535;
        hipLaunchKernelGGL((k_kv_weigh_again<T, CH>), dim3(few.units * a.pairs, z), dim3(256), 0, stream, a);
    }
    return true;
}

template <typename T>
int run_attend(const Attend& a, const Cut& k, bool accumulate, hipStream_t stream)
{
    bool ok = false;
    switch (a.c.dims / 64) {
    case 1: ok = launch_attend<T, 1>(a, k, accumulate, stream); break;
    case 2: ok = launch_attend<T, 2>(a, k, accumulate, stream); break;
    case 3: ok = launch_attend<T, 3>(a, k, accumulate, stream); break;
    default: ok = launch_attend<T, 4>(a, k, accumulate, stream); break;
    }
    return ok ? checked(hipGetLastError()) : HBFSIM_CUDA_ERROR;
}

}  // namespace

#define HBF_API extern "C" __attribute__((visibility("default")))

HBF_API int hbfsim_amd_kv_append(const hbfsim_amd_kv_cache* cache, const hbfsim_amd_kv_batch* batch,
                                 const void* d_k, const void* d_v, uint32_t type,
                                 const int64_t strides[4], void* stream)
{
    Append a{};
    int rc = take_cache(cache, &a.c);
    if (rc == HBFSIM_OK) rc = take_batch(batch, a.c, &a.b);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    if (type > HBFSIM_AMD_KV_F32 || strides == nullptr) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (a.b.tokens == 0 || a.b.seqs == 0 || a.b.width == 0) {
        return HBFSIM_OK;
    }
    if (d_k == nullptr || d_v == nullptr) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    a.x[0] = d_k;
    a.x[1] = d_v;
    for (int i = 0; i < 2; ++i) {
        a.token_stride[i] = strides[2 * i];
        a.head_stride[i] = strides[2 * i + 1];
    }
    const std::uint64_t blocks = a.b.first == nullptr ? a.b.seqs : a.b.tokens / a.c.tokens + std::uint64_t{2} * a.b.seqs;
    if (blocks > kMostGroups) {
        return HBFSIM_UNSUPPORTED;
    }
    const std::uint32_t slots = static_cast<std::uint32_t>(blocks);
    const std::size_t each = type == HBFSIM_AMD_KV_F32 ? 4 : 8;  // elements of 16 bytes
    for (int i = 0; i < 2; ++i) {
        a.vector[i] = aligned16(a.x[i]) && a.token_stride[i] % static_cast<std::int64_t>(each) == 0 &&
                              a.head_stride[i] % static_cast<std::int64_t>(each) == 0
                          ? 1
                          : 0;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == HBFSIM_AMD_KV_BF16) {
        run_append<Bf16>(a, slots, s);
    } else if (type == HBFSIM_AMD_KV_F16) {
        run_append<F16>(a, slots, s);
    } else {
        run_append<float>(a, slots, s);
    }
    return checked(hipGetLastError());
}

HBF_API int hbfsim_amd_kv_read(const hbfsim_amd_kv_cache* cache, const int32_t* d_blocks, size_t n,
                               uint32_t type, void* d_k, void* d_v, void* d_low, void* d_high,
                               void* stream)
{
    Cache c{};
    const int rc = take_cache(cache, &c);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    if (type > HBFSIM_AMD_KV_F32) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (n > kMostGroups) {
        return HBFSIM_UNSUPPORTED;
    }
    if (n == 0) {
        return HBFSIM_OK;
    }
    if (d_blocks == nullptr || d_k == nullptr || d_v == nullptr || d_low == nullptr || d_high == nullptr) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const std::uint32_t vector = aligned16(d_k) && aligned16(d_v) ? 1 : 0, count = static_cast<std::uint32_t>(n);
    if (type == HBFSIM_AMD_KV_BF16) {
        run_read<Bf16>(c, d_blocks, count, d_k, d_v, d_low, d_high, vector, s);
    } else if (type == HBFSIM_AMD_KV_F16) {
        run_read<F16>(c, d_blocks, count, d_k, d_v, d_low, d_high, vector, s);
    } else {
        run_read<float>(c, d_blocks, count, d_k, d_v, d_low, d_high, vector, s);
    }
    return checked(hipGetLastError());
}

HBF_API int hbfsim_amd_kv_attend_workspace(const hbfsim_amd_kv_cache* cache, const hbfsim_amd_kv_batch* batch,
                                           uint32_t heads, uint32_t count, uint32_t accumulate, size_t* bytes)
{
    Cache c{};
    Batch b{};
    int rc = take_cache(cache, &c);
    if (rc == HBFSIM_OK) rc = take_batch(batch, c, &b);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    if (bytes == nullptr || heads == 0 || heads % c.kv_heads != 0) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    *bytes = b.tokens == 0 || b.seqs == 0 ? 0 : cut_attend(c, b, heads, count, accumulate != 0).bytes;
    return HBFSIM_OK;
}

HBF_API int hbfsim_amd_kv_attend(const hbfsim_amd_kv_cache* cache, const hbfsim_amd_kv_batch* batch,
                                 const void* d_q, uint32_t type, uint32_t heads, int64_t token_stride,
                                 int64_t head_stride, float scale, const int32_t* d_selected, uint32_t count,
                                 uint32_t accumulate, void* d_out, void* d_workspace, size_t workspace_bytes,
                                 void* stream)
{
    Attend a{};
    int rc = take_cache(cache, &a.c);
    if (rc == HBFSIM_OK) rc = take_batch(batch, a.c, &a.b);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    if (!two_byte(type) || heads == 0 || heads % a.c.kv_heads != 0 || !(scale == scale) ||
        scale == kInf || scale == -kInf || (d_selected == nullptr) != (count == 0) ||
        (accumulate != 0 && count != 0) || static_cast<std::uint64_t>(count) * a.c.tokens > 0x7fffff00u) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (a.b.tokens == 0) {
        return HBFSIM_OK;
    }
    Cut k{};
    if (a.b.seqs != 0) k = cut_attend(a.c, a.b, heads, count, accumulate != 0);
    if (d_q == nullptr || d_out == nullptr || workspace_bytes < k.bytes ||
        (k.bytes != 0 && (d_workspace == nullptr || !aligned16(d_workspace)))) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    // weights of several tokens a sequence may read the queries a second time
    bool same = false;
    if (overlaps(reinterpret_cast<std::uintptr_t>(d_q), token_stride, head_stride, reinterpret_cast<std::uintptr_t>(d_out),
                 a.b.tokens, heads, a.c.dim, &same) &&
        (!same || (accumulate != 0 && a.b.first != nullptr))) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    const Cut few = cut_few(a.c, a.b, heads, count);
    if (static_cast<std::uint64_t>(k.units) * a.c.kv_heads * k.row_tiles > kMostGroups || k.splits > 65535 ||
        (accumulate != 0 && (static_cast<std::uint64_t>(few.units) * a.c.kv_heads * few.row_tiles > kMostGroups ||
                             a.b.width > 65535 * 256u))) {
        return HBFSIM_UNSUPPORTED;
    }
    a.q = d_q;
    a.q_token = token_stride;
    a.q_head = head_stride;
    a.q_vector = aligned16(d_q) && token_stride % 8 == 0 && head_stride % 8 == 0 ? 1 : 0;
    a.out_vector = (reinterpret_cast<std::uintptr_t>(d_out) & 7u) == 0 ? 1 : 0;
    a.heads = heads;
    a.group = heads / a.c.kv_heads;
    a.per = k.per;
    a.row_tiles = k.row_tiles;
    a.rows = k.rows;
    a.pairs = a.c.kv_heads * k.row_tiles;
    a.scale = scale * kLog2e;
    a.selected = d_selected;
    a.count = count;
    a.split = k.split;
    a.splits = k.splits;
    a.out = d_out;
    unsigned char* ws = static_cast<unsigned char*>(d_workspace);
    a.partial = k.splits > 1 ? reinterpret_cast<float*>(ws + k.partial) : nullptr;
    a.stats = k.splits > 1 ? reinterpret_cast<float*>(ws + k.stats) : nullptr;
    a.lse = accumulate != 0 ? reinterpret_cast<float*>(ws + k.lse) : nullptr;
    a.tile_sums = accumulate != 0 && k.many == 0 ? reinterpret_cast<float*>(ws + k.tile_sums) : nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return type == HBFSIM_AMD_KV_BF16 ? run_attend<Bf16>(a, k, accumulate != 0, s)
                                      : run_attend<F16>(a, k, accumulate != 0, s);
}

HBF_API int hbfsim_amd_kv_select_workspace(const hbfsim_amd_kv_cache* cache, const hbfsim_amd_kv_batch* batch,
                                           size_t* bytes)
{
    Cache c{};
    Batch b{};
    int rc = take_cache(cache, &c);
    if (rc == HBFSIM_OK) rc = take_batch(batch, c, &b);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    if (bytes == nullptr) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    *bytes = select_bytes(c, b);
    return HBFSIM_OK;
}

HBF_API int hbfsim_amd_kv_select(const hbfsim_amd_kv_cache* cache, const hbfsim_amd_kv_batch* batch,
                                 const void* d_q, uint32_t type, uint32_t heads, int64_t token_stride,
                                 int64_t head_stride, uint32_t count, uint32_t keep_first, uint32_t keep_last,
                                 int32_t* d_selected, void* d_workspace, size_t workspace_bytes, void* stream)
{
    Select a{};
    int rc = take_cache(cache, &a.c);
    if (rc == HBFSIM_OK) rc = take_batch(batch, a.c, &a.b);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    if (!two_byte(type) || heads == 0 || heads % a.c.kv_heads != 0 || heads / a.c.kv_heads > 64 || count == 0 ||
        count > 0x7fffffffu || static_cast<std::uint64_t>(keep_first) + keep_last > count) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (a.b.tokens == 0) {
        return HBFSIM_OK;
    }
    const bool one = select_in_one(a.c, a.b);
    const std::size_t need = select_bytes(a.c, a.b);
    if (d_q == nullptr || d_selected == nullptr || workspace_bytes < need ||
        (need != 0 && (d_workspace == nullptr || !aligned16(d_workspace)))) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    // scores come in workgroups of a quarter of the threads
    if (static_cast<std::uint64_t>(a.b.tokens) * a.c.kv_heads > kMostGroups ||
        (!one && static_cast<std::uint64_t>(score_slots(a.b)) * a.c.kv_heads > 4 * kMostGroups)) {
        return HBFSIM_UNSUPPORTED;
    }
    a.q = d_q;
    a.q_token = token_stride;
    a.q_head = head_stride;
    a.group = heads / a.c.kv_heads;
    a.count = count;
    a.keep_first = keep_first;
    a.keep_last = keep_last;
    a.keys = static_cast<std::uint32_t*>(d_workspace);
    a.selected = d_selected;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    bool ok = true;
    if (type == HBFSIM_AMD_KV_BF16) {
        ok = run_select<Bf16>(a, one, s);
    } else {
        ok = run_select<F16>(a, one, s);
    }
    return ok ? checked(hipGetLastError()) : HBFSIM_CUDA_ERROR;
}

HBF_API int hbfsim_amd_kv_evict(const int64_t* d_weight, uint32_t blocks, uint32_t kv_heads, uint32_t block_tokens,
                                const int32_t* d_table, const int32_t* d_lens, uint32_t seqs, uint32_t width,
                                uint32_t stride, uint32_t keep, uint32_t keep_first, uint32_t keep_last,
                                int32_t* d_out_table, int32_t* d_out_lens, int32_t* d_freed,
                                int32_t* d_freed_count, void* d_workspace, size_t workspace_bytes, void* stream)
{
    const bool tokens_ok = block_tokens == 16 || block_tokens == 32 || block_tokens == 64 || block_tokens == 128;
    if (blocks == 0 || blocks > 0x7fffffffu || kv_heads == 0 || kv_heads > 1024 || !tokens_ok || keep == 0 ||
        keep_last == 0 || static_cast<std::uint64_t>(keep_first) + keep_last > keep || stride < width ||
        seqs > 0x7fffff00u || static_cast<std::uint64_t>(width) * block_tokens > 0x7fffff00u) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (seqs == 0) {
        return HBFSIM_OK;
    }
    if (seqs > kMostGroups) {
        return HBFSIM_UNSUPPORTED;
    }
    const std::size_t need = static_cast<std::size_t>(seqs) * width * sizeof(unsigned long long);
    if (d_weight == nullptr || d_lens == nullptr || d_out_lens == nullptr || d_freed_count == nullptr ||
        workspace_bytes < need || (need != 0 && (d_table == nullptr || d_out_table == nullptr || d_freed == nullptr ||
                                                 d_workspace == nullptr || !aligned16(d_workspace)))) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    Evict a{reinterpret_cast<const unsigned long long*>(d_weight), blocks, kv_heads, block_tokens, d_table, d_lens,
            seqs, width, stride, keep, keep_first, keep_last, static_cast<unsigned long long*>(d_workspace),
            d_out_table, d_out_lens, d_freed, d_freed_count};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const std::size_t lds = static_cast<std::size_t>(width) * sizeof(unsigned long long);
    if (lds <= kMostStaged) {
        if (!lds_allowed(reinterpret_cast<const void*>(&k_kv_evict<true>), lds)) {
            return HBFSIM_CUDA_ERROR;
        }
        hipLaunchKernelGGL(k_kv_evict<true>, dim3(seqs), dim3(kPickThreads), lds, s, a);
    } else {
        hipLaunchKernelGGL(k_kv_evict<false>, dim3(seqs), dim3(kPickThreads), 0, s, a);
    }
    return checked(hipGetLastError());
}
