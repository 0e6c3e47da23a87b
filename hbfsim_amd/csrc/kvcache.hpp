// kvcache.hpp -- what the paged cache's operators share: a call's view of the
// cache and the batch, its checks, and how a wave finds a sequence.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/hbfsim_amd.h"

#include <cstddef>
#include <cstdint>

namespace hbfamd {
namespace kv {

constexpr int kWave = 64;

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

// ---- host -----------------------------------------------------------------

// A launch dimension holds fewer than 2^32 threads, a workgroup at most 1024.
constexpr std::size_t kMostGroups = (std::size_t{1} << 22) - 1;

inline bool aligned16(const void* p) { return (reinterpret_cast<std::uintptr_t>(p) & 15u) == 0; }

inline int checked(hipError_t e) { return e == hipSuccess ? HBFSIM_OK : HBFSIM_CUDA_ERROR; }

// The cache's own fields; pools may be asked for or not.
inline int take_cache(const hbfsim_amd_kv_cache* in, Cache* out)
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

inline int take_batch(const hbfsim_amd_kv_batch* in, const Cache& c, Batch* out)
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

// Whether [p, p + n) and [q, q + m) have a byte in common.
inline bool meet(const void* p, std::size_t n, const void* q, std::size_t m)
{
    const std::uintptr_t a = reinterpret_cast<std::uintptr_t>(p), b = reinterpret_cast<std::uintptr_t>(q);
    return p != nullptr && q != nullptr && n != 0 && m != 0 && a < b + m && b < a + n;
}

inline std::size_t up256(std::size_t x) { return (x + 255) & ~std::size_t{255}; }

}  // namespace kv
}  // namespace hbfamd
