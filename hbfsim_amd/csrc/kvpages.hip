// kvpages.hip -- the blocks of branching sequences: who holds them, and moves
// of their contents: copy, hold, fork, release, grow, compact.
//
// No counterpart in the reference.  A count per block says how many table
// entries name it; the operators change counts and entries together, so that a
// step that branches, grows and gives back blocks never asks the host.  Counts
// are whole numbers and every choice is by sequence, place and id, so results
// do not depend on which workgroup is first.
#include "kvcache.hpp"

namespace {

using namespace hbfamd::kv;

constexpr int kThreads = 256;

__device__ inline bool inside(std::int32_t id, std::uint32_t blocks) { return static_cast<std::uint32_t>(id) < blocks; }

// ---- contents ---------------------------------------------------------------

// What a block holds, in units of 16 bytes: keys, values, bounds; then floats
// and weights of each kv head.
struct Piece {
    std::uint32_t codes, bounds;  // units of keys (as many of values), and of bounds
    std::uint32_t parts, per;     // workgroups per block, units of each (a multiple of 64)
};

// One workgroup's part of a block.  A wave's 64 units are of one array, as a
// block's keys and values are whole KiB.
__device__ inline void copy_part(const Cache& from, const Cache& to, const Piece& p, std::int32_t src, std::int32_t dst,
                                 std::uint32_t part)
{
    const std::uint32_t all = 2 * p.codes + p.bounds;
    const std::uint32_t end = (part + 1) * p.per < all ? (part + 1) * p.per : all;
    const std::size_t s = static_cast<std::size_t>(src), d = static_cast<std::size_t>(dst);
    const u32x4* keys = reinterpret_cast<const u32x4*>(from.keys) + s * p.codes;
    const u32x4* values = reinterpret_cast<const u32x4*>(from.values) + s * p.codes;
    const u32x4* bounds = reinterpret_cast<const u32x4*>(from.bounds) + s * p.bounds;
    u32x4* keys_to = reinterpret_cast<u32x4*>(to.keys) + d * p.codes;
    u32x4* values_to = reinterpret_cast<u32x4*>(to.values) + d * p.codes;
    u32x4* bounds_to = reinterpret_cast<u32x4*>(to.bounds) + d * p.bounds;
    for (std::uint32_t i = part * p.per + threadIdx.x; i < end; i += kThreads) {
        if (i < p.codes) {
            keys_to[i] = keys[i];
        } else if (i < 2 * p.codes) {
            values_to[i - p.codes] = values[i - p.codes];
        } else {
            bounds_to[i - 2 * p.codes] = bounds[i - 2 * p.codes];
        }
    }
    if (part == 0) {
        for (std::uint32_t h = threadIdx.x; h < from.kv_heads; h += kThreads) {
            to.key_scale[d * from.kv_heads + h] = from.key_scale[s * from.kv_heads + h];
            to.value_scale[d * from.kv_heads + h] = from.value_scale[s * from.kv_heads + h];
            to.weight[d * from.kv_heads + h] = from.weight[s * from.kv_heads + h];
        }
    }
}

struct Copy {
    Cache from, to;
    Piece p;
    const std::int32_t* src;
    const std::int32_t* dst;
    std::uint32_t n, same;
    std::int32_t* owner;  // [to.blocks]: the first pair that names the block as its destination
};
constexpr std::int32_t kNobody = 0x7fffffff;

__device__ inline bool pair_at(const Copy& a, std::uint32_t i, std::int32_t* src, std::int32_t* dst)
{
    *src = a.src[i];
    *dst = a.dst[i];
    return inside(*src, a.from.blocks) && inside(*dst, a.to.blocks);
}
__global__ __launch_bounds__(kThreads) void k_kv_copy_clear(Copy a)
{
    const std::uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    std::int32_t src, dst;
    if (i < a.n && pair_at(a, i, &src, &dst)) {
        a.owner[dst] = kNobody;
        if (a.same != 0) a.owner[src] = kNobody;
    }
}
__global__ __launch_bounds__(kThreads) void k_kv_copy_claim(Copy a)
{
    const std::uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    std::int32_t src, dst;
    if (i < a.n && pair_at(a, i, &src, &dst)) atomicMin(&a.owner[dst], static_cast<std::int32_t>(i));
}
// A destination that an invalid pair names is claimed by nobody: pairs count
// only where both ids are of their pools.
__global__ __launch_bounds__(kThreads) void k_kv_copy(Copy a)
{
    const std::uint32_t i = blockIdx.x / a.p.parts, part = blockIdx.x % a.p.parts;
    std::int32_t src, dst;
    if (!pair_at(a, i, &src, &dst) || a.owner[dst] != static_cast<std::int32_t>(i) ||
        (a.same != 0 && a.owner[src] != kNobody)) {
        return;
    }
    copy_part(a.from, a.to, a.p, src, dst, part);
}

// ---- counts and tables --------------------------------------------------------

struct Table {
    std::int32_t* refs;
    std::uint32_t blocks, tokens;
    std::int32_t* table;
    const std::int32_t* lens;
    std::uint32_t seqs, width, stride;
    std::uint32_t chunks;  // workgroups per row
};
constexpr std::uint32_t kRow = kThreads * 4;  // entries of a workgroup

template <typename F>
__device__ inline void each_entry(const Table& a, std::uint32_t chunk, F f)
{
#pragma unroll
    for (std::uint32_t k = 0; k < kRow; k += kThreads) {
        const std::uint32_t i = chunk * kRow + k + threadIdx.x;
        if (i < a.width) f(i);
    }
}

__global__ __launch_bounds__(kThreads) void k_kv_hold(Table a)
{
    const std::uint32_t s = blockIdx.x / a.chunks;
    const std::int32_t* row = a.table + static_cast<std::size_t>(s) * a.stride;
    each_entry(a, blockIdx.x % a.chunks, [&](std::uint32_t i) {
        const std::int32_t id = row[i];
        if (inside(id, a.blocks)) atomicAdd(&a.refs[id], 1);
    });
}

__global__ __launch_bounds__(kThreads) void k_kv_release(Table a)
{
    const std::uint32_t s = blockIdx.x / a.chunks;
    std::int32_t* row = a.table + static_cast<std::size_t>(s) * a.stride;
    const std::int64_t len = a.lens == nullptr || a.lens[s] < 0 ? 0 : a.lens[s];
    const std::int64_t keep = (len + a.tokens - 1) / a.tokens;
    each_entry(a, blockIdx.x % a.chunks, [&](std::uint32_t i) {
        if (static_cast<std::int64_t>(i) < keep) return;
        const std::int32_t id = row[i];
        if (inside(id, a.blocks)) atomicSub(&a.refs[id], 1);
        if (id != -1) row[i] = -1;
    });
}

struct Fork {
    Table t;
    const std::int32_t* parents;
    std::uint32_t rows;
    std::int32_t* out;
    std::int32_t* out_lens;
};
// The first rows * chunks workgroups write the new rows, the others change the
// old rows' counts by their children less one.
__global__ __launch_bounds__(kThreads) void k_kv_fork(Fork a)
{
    const std::uint32_t r = blockIdx.x / a.t.chunks, chunk = blockIdx.x % a.t.chunks;
    if (r < a.rows) {
        const std::int32_t p = a.parents[r];
        const bool there = inside(p, a.t.seqs);
        const std::int32_t* row = a.t.table + static_cast<std::size_t>(there ? p : 0) * a.t.stride;
        each_entry(a.t, chunk, [&](std::uint32_t i) { a.out[static_cast<std::size_t>(r) * a.t.width + i] = there ? row[i] : -1; });
        if (chunk == 0 && threadIdx.x == 0) a.out_lens[r] = there ? a.t.lens[p] : 0;
        return;
    }
    const std::uint32_t s = r - a.rows;
    __shared__ std::int32_t s_count[kThreads / kWave];
    std::int32_t children = 0;
    for (std::uint32_t i = threadIdx.x; i < a.rows; i += kThreads) children += a.parents[i] == static_cast<std::int32_t>(s);
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) children += __shfl_xor(children, k);
    if (threadIdx.x % kWave == 0) s_count[threadIdx.x / kWave] = children;
    __syncthreads();
    children = 0;
#pragma unroll
    for (int i = 0; i < kThreads / kWave; ++i) children += s_count[i];
    if (children == 1) {
        return;
    }
    const std::int32_t* row = a.t.table + static_cast<std::size_t>(s) * a.t.stride;
    each_entry(a.t, chunk, [&](std::uint32_t i) {
        const std::int32_t id = row[i];
        if (inside(id, a.t.blocks)) atomicAdd(&a.t.refs[id], children - 1);
    });
}

// ---- grow -------------------------------------------------------------------

constexpr int kPlan = 1024;  // threads of the workgroup that plans
constexpr int kPlanWaves = kPlan / kWave;

struct Grow {
    Cache c;
    Piece p;
    std::int32_t* refs;
    std::int32_t* table;
    const std::int32_t* lens;
    const std::int32_t* first;
    std::uint32_t seqs, tokens, width, stride, slots;
    std::int32_t* out_lens;
    std::int32_t* missing;
    // workspace
    std::int32_t* need;     // [slots + 1]: new blocks of the slots before
    int4* slot;             // [slots]: sequence, place, the row's block or what to do without
    std::int32_t* found;    // [slots]: free blocks, ascending
    std::int32_t* writers;  // [blocks]: slots that write to a shared block, and the last of them
    std::int32_t* last;
    int2* pair;             // [seqs]: content to copy, source and destination
};
constexpr std::int32_t kNew = -1;    // no block of its own: a new one
constexpr std::int32_t kIdle = -2;   // nothing to do
constexpr std::int32_t kStale = -3;  // a begun block that is free

// A sequence's part of the step: tokens [from, to) of its own, none if the
// offsets do not describe the batch.
struct Part {
    std::int64_t from, to;
};
__device__ inline Part part_of(const Grow& a, std::uint32_t s)
{
    const std::int64_t to = a.lens[s];
    std::int64_t begin = s, count = 1;
    if (a.first != nullptr) {
        begin = a.first[s];
        count = a.first[s + 1] - begin;
    }
    if (count <= 0 || begin < 0 || begin + count > a.tokens || to < count) {
        return Part{0, 0};
    }
    return Part{to - count, to};
}
// Sequence s owns the slots from floor(first[s] / t) + 2 s on.
__device__ inline std::uint32_t base_of(const Grow& a, std::uint32_t s)
{
    if (a.first == nullptr) return s;
    const std::uint64_t at = static_cast<std::uint32_t>(a.first[s]) / a.c.tokens + std::uint64_t{2} * s;
    return at < a.slots ? static_cast<std::uint32_t>(at) : a.slots;
}
__device__ inline std::int32_t now(const std::int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ inline void settled()  // what the workgroup stored is seen by all of it
{
    __threadfence();
    __syncthreads();
}

// Sums before each thread's `x`, and of all; all threads call it.
__device__ inline std::int32_t before(std::int32_t x, std::int32_t* all)
{
    __shared__ std::int32_t s_wave[kPlanWaves];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    std::int32_t upto = x;
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) {
        const std::int32_t y = __shfl_up(upto, k);
        upto += lane >= k ? y : 0;
    }
    __syncthreads();
    if (lane == kWave - 1) s_wave[wave] = upto;
    __syncthreads();
    std::int32_t sum = 0;
    upto -= x;
#pragma unroll
    for (int i = 0; i < kPlanWaves; ++i) {
        upto += i < wave ? s_wave[i] : 0;
        sum += s_wave[i];
    }
    *all = sum;
    return upto;
}

// Writes need[]; returns the new blocks of all slots.
template <typename F>
__device__ inline std::int32_t count_needs(const Grow& a, F fresh)
{
    std::int32_t total = 0;
    for (std::uint32_t base = 0; base < a.slots; base += kPlan) {
        const std::uint32_t i = base + threadIdx.x;
        std::int32_t all;
        const std::int32_t at = before(i < a.slots && fresh(i) ? 1 : 0, &all);
        if (i < a.slots) a.need[i] = total + at;
        total += all;
    }
    if (threadIdx.x == 0) a.need[a.slots] = total;
    settled();
    return total;
}

__global__ __launch_bounds__(kPlan) void k_kv_grow(Grow a)
{
    const std::uint32_t t = a.c.tokens;
    // what each slot writes to
    bool shared = false;
    for (std::uint32_t i = threadIdx.x; i < a.slots; i += kPlan) {
        std::uint32_t s = i;
        if (a.first != nullptr) {
            std::uint32_t lo = 0, hi = a.seqs;  // the last sequence whose slots begin at or before i
            while (hi - lo > 1) {
                const std::uint32_t mid = lo + (hi - lo) / 2;
                if (base_of(a, mid) <= i) lo = mid; else hi = mid;
            }
            s = lo;
        }
        int4 slot = {static_cast<int>(s), 0, kIdle, 0};
        const Part part = part_of(a, s);
        const std::uint32_t base = base_of(a, s);
        const std::int64_t place = part.from / t + (static_cast<std::int64_t>(i) - base);
        if (i >= base && place * t < part.to && (part.to - 1) / t < static_cast<std::int64_t>(a.width)) {
            const std::int32_t id = a.table[static_cast<std::size_t>(s) * a.stride + place];
            const bool named = inside(id, a.c.blocks), begun = place * t < part.from;
            const std::int32_t refs = named ? a.refs[id] : 0;
            slot.y = static_cast<int>(place);
            if (refs > 0) {
                slot.z = id;
                slot.w = refs;
                if (refs > 1) {
                    shared = true;
                    a.writers[id] = 0;
                    a.last[id] = -1;
                }
            } else {
                slot.z = !begun ? kNew : named ? kStale : kIdle;
            }
        }
        a.slot[i] = slot;
    }
    for (std::uint32_t s = threadIdx.x; s < a.seqs; s += kPlan) a.pair[s] = int2{-1, -1};
    const bool any = __syncthreads_or(shared);
    if (any) {
        settled();
        for (std::uint32_t i = threadIdx.x; i < a.slots; i += kPlan) {
            const int4 slot = a.slot[i];
            if (slot.z >= 0 && slot.w > 1) {
                atomicAdd(&a.writers[slot.z], 1);
                atomicMax(&a.last[slot.z], static_cast<std::int32_t>(i));
            }
        }
    }
    settled();
    const auto keeps = [&](std::uint32_t i) {
        const int4 slot = a.slot[i];
        return slot.w <= 1 || (now(&a.writers[slot.z]) >= slot.w && now(&a.last[slot.z]) == static_cast<std::int32_t>(i));
    };
    const auto fresh = [&](std::uint32_t i) {
        const int z = a.slot[i].z;
        return z == kNew || (z >= 0 && !keeps(i));
    };
    const auto fresh_alone = [&](std::uint32_t i) {  // no shared block is kept
        const int4 slot = a.slot[i];
        return slot.z == kNew || (slot.z >= 0 && slot.w > 1);
    };
    std::int32_t want = count_needs(a, fresh);
    // free blocks, as many as are wanted
    std::int32_t free = 0;
    for (std::uint64_t at = 0; at < a.c.blocks && free < want; at += kPlan) {
        const std::uint64_t id = at + threadIdx.x;
        const bool is = id < a.c.blocks && a.refs[id] <= 0;
        std::int32_t all;
        const std::int32_t rank = free + before(is ? 1 : 0, &all);
        if (is && rank < want) a.found[rank] = static_cast<std::int32_t>(id);
        free += all;
    }
    const bool enough = free >= want;
    if (!enough) want = count_needs(a, fresh_alone);
    settled();
    const auto granted = [&](std::uint32_t s) {
        const Part part = part_of(a, s);
        if (part.to > 0 && (part.to - 1) / t >= static_cast<std::int64_t>(a.width)) return false;
        const std::int32_t from = a.need[base_of(a, s)], to = a.need[s + 1 < a.seqs ? base_of(a, s + 1) : a.slots];
        return enough || to == from || to <= free;
    };
    for (std::uint32_t i = threadIdx.x; i < a.slots; i += kPlan) {
        const int4 slot = a.slot[i];
        if (slot.z == kIdle || !granted(slot.x)) continue;
        std::int32_t* entry = a.table + static_cast<std::size_t>(slot.x) * a.stride + slot.y;
        if (slot.z == kStale) {
            *entry = -1;
        } else if (enough ? fresh(i) : fresh_alone(i)) {
            const std::int32_t id = a.found[a.need[i]];
            *entry = id;
            a.refs[id] = 1;
            if (slot.z >= 0) {
                atomicSub(&a.refs[slot.z], 1);
                if (static_cast<std::int64_t>(slot.y) * t < part_of(a, slot.x).from) a.pair[slot.x] = int2{slot.z, id};
            }
        }
    }
    __syncthreads();  // the lengths may become the new ones
    for (std::uint32_t s = threadIdx.x; s < a.seqs; s += kPlan) {
        const Part part = part_of(a, s);
        std::int32_t lacks = 0;
        if (!granted(s)) {
            const std::int64_t from = part.from / t, to = (part.to - 1) / t + 1, width = a.width;
            lacks = to > width ? static_cast<std::int32_t>(to - (from > width ? from : width))
                               : a.need[s + 1 < a.seqs ? base_of(a, s + 1) : a.slots] - a.need[base_of(a, s)];
        }
        a.missing[s] = lacks;
        a.out_lens[s] = lacks != 0 ? 0 : a.lens[s];
    }
}

__global__ __launch_bounds__(kThreads) void k_kv_grow_copy(Grow a)
{
    const int2 pair = a.pair[blockIdx.x / a.p.parts];
    if (pair.x >= 0) copy_part(a.c, a.c, a.p, pair.x, pair.y, blockIdx.x % a.p.parts);
}

// ---- compact ------------------------------------------------------------------

constexpr std::uint32_t kChunk = kThreads * 4;  // blocks of a workgroup

struct Compact {
    Cache c;
    Piece p;
    Table t;
    std::int32_t* where;
    std::uint32_t chunks;
    std::uint32_t* count;  // [chunks]: blocks in use
    std::uint32_t* moves;  // how many
    std::int32_t* source;  // [blocks / 2]: the j-th block in use past the front
    std::int32_t* hole;    // [blocks / 2]: the j-th free one of the front
};
constexpr std::int32_t kMoves = -2;  // where: minus the rank of the move

template <typename T>
__device__ inline T sum_all(T x)  // over the workgroup, for all of it
{
    __shared__ T s_sum[kThreads / kWave];
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) x += __shfl_xor(x, k);
    __syncthreads();
    if (threadIdx.x % kWave == 0) s_sum[threadIdx.x / kWave] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int i = 0; i < kThreads / kWave; ++i) x += s_sum[i];
    return x;
}

__device__ inline std::uint32_t in_use(const Compact& a, std::uint32_t id) { return id < a.c.blocks && a.t.refs[id] > 0 ? 1 : 0; }

__global__ __launch_bounds__(kThreads) void k_kv_compact_count(Compact a)
{
    std::uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) mine += in_use(a, blockIdx.x * kChunk + k * kThreads + threadIdx.x);
    mine = sum_all(mine);
    if (threadIdx.x == 0) a.count[blockIdx.x] = mine;
}

__global__ __launch_bounds__(kThreads) void k_kv_compact_plan(Compact a)
{
    __shared__ std::uint32_t s_wave[kThreads / kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    std::uint32_t earlier = 0, live = 0;
    for (std::uint32_t i = threadIdx.x; i < a.chunks; i += kThreads) {
        const std::uint32_t n = a.count[i];
        live += n;
        earlier += i < blockIdx.x ? n : 0;
    }
    live = sum_all(live);
    earlier = sum_all(earlier);
    // blocks in use before the front's end
    std::uint32_t front = 0;
    for (std::uint32_t i = threadIdx.x; i < live / kChunk; i += kThreads) front += a.count[i];
    for (std::uint32_t i = live / kChunk * kChunk + threadIdx.x; i < live; i += kThreads) front += in_use(a, i);
    front = sum_all(front);
    std::uint32_t used[4], mine = 0;
    const std::uint32_t id0 = blockIdx.x * kChunk + threadIdx.x * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        used[k] = in_use(a, id0 + k);
        mine += used[k];
    }
    std::uint32_t upto = mine;
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) {
        const std::uint32_t y = __shfl_up(upto, k);
        upto += lane >= k ? y : 0;
    }
    if (lane == kWave - 1) s_wave[wave] = upto;
    __syncthreads();
    std::uint32_t at = earlier + upto - mine;  // blocks in use before this one
#pragma unroll
    for (int i = 0; i < kThreads / kWave; ++i) at += i < wave ? s_wave[i] : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const std::uint32_t id = id0 + k;
        if (id < a.c.blocks) {
            std::int32_t to = -1;
            if (used[k] != 0) {
                to = static_cast<std::int32_t>(id);
                if (id >= live) {
                    a.source[at - front] = static_cast<std::int32_t>(id);
                    to = kMoves - static_cast<std::int32_t>(at - front);
                }
            } else if (id < live) {
                a.hole[id - at] = static_cast<std::int32_t>(id);
            }
            a.where[id] = to;
        }
        at += used[k];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.moves = live - front;
}

// The first workgroups move blocks, those from `movers` on the table's entries.
// An entry's block may get its place in `where` meanwhile: either form says it.
__global__ __launch_bounds__(kThreads) void k_kv_compact(Compact a, std::uint32_t movers)
{
    if (blockIdx.x >= movers) {
        const std::uint32_t s = (blockIdx.x - movers) / a.t.chunks;
        std::int32_t* row = a.t.table + static_cast<std::size_t>(s) * a.t.stride;
        each_entry(a.t, (blockIdx.x - movers) % a.t.chunks, [&](std::uint32_t i) {
            const std::int32_t id = row[i];
            std::int32_t to = inside(id, a.c.blocks) ? now(&a.where[id]) : -1;
            if (to <= kMoves) to = a.hole[kMoves - to];
            if (to != id) row[i] = to;
        });
        return;
    }
    const std::uint64_t items = static_cast<std::uint64_t>(*a.moves) * a.p.parts;
    for (std::uint64_t i = blockIdx.x; i < items; i += movers) {
        const std::uint32_t j = static_cast<std::uint32_t>(i / a.p.parts), part = static_cast<std::uint32_t>(i % a.p.parts);
        const std::int32_t src = a.source[j], dst = a.hole[j];
        copy_part(a.c, a.c, a.p, src, dst, part);
        if (part == 0 && threadIdx.x == 0) {
            a.t.refs[dst] = a.t.refs[src];
            a.t.refs[src] = 0;
            __hip_atomic_store(&a.where[src], dst, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// ---- host -----------------------------------------------------------------

constexpr std::uint64_t kMostWork = 4 * kMostGroups;  // workgroups of kThreads in a launch

Piece piece_of(const Cache& c)
{
    Piece p{};
    p.codes = c.kv_heads * c.tokens * c.dims / 16;
    p.bounds = c.kv_heads * 2 * c.dims / 16;
    const std::uint32_t all = 2 * p.codes + p.bounds;
    p.parts = (all + 4 * kThreads - 1) / (4 * kThreads);
    p.per = ((all + p.parts - 1) / p.parts + kWave - 1) / kWave * kWave;
    return p;
}

std::size_t block_bytes(const Cache& c) { return static_cast<std::size_t>(c.kv_heads) * c.tokens * c.dims; }

// Whether [p, p + n) and [q, q + m) have a byte in common.
bool meet(const void* p, std::size_t n, const void* q, std::size_t m)
{
    const std::uintptr_t a = reinterpret_cast<std::uintptr_t>(p), b = reinterpret_cast<std::uintptr_t>(q);
    return n != 0 && m != 0 && a < b + m && b < a + n;
}

// Two caches share nothing.
bool apart(const Cache& x, const Cache& y)
{
    const std::size_t nx = x.blocks, ny = y.blocks, heads = x.kv_heads, codes = block_bytes(x);
    return !meet(x.keys, nx * codes, y.keys, ny * codes) && !meet(x.values, nx * codes, y.values, ny * codes) &&
           !meet(x.bounds, nx * heads * 2 * x.dims, y.bounds, ny * heads * 2 * y.dims) &&
           !meet(x.key_scale, nx * heads * 4, y.key_scale, ny * heads * 4) &&
           !meet(x.value_scale, nx * heads * 4, y.value_scale, ny * heads * 4) &&
           !meet(x.weight, nx * heads * 8, y.weight, ny * heads * 8);
}
bool same(const Cache& x, const Cache& y)
{
    return x.keys == y.keys && x.values == y.values && x.bounds == y.bounds && x.key_scale == y.key_scale &&
           x.value_scale == y.value_scale && x.weight == y.weight && x.blocks == y.blocks;
}

int take_table(std::int32_t* refs, std::uint32_t blocks, std::uint32_t tokens, std::int32_t* table, std::uint32_t seqs,
               std::uint32_t width, std::uint32_t stride, Table* out)
{
    if (refs == nullptr || blocks == 0 || blocks > 0x7fffffffu || stride < width || seqs > 0x7fffff00u ||
        static_cast<std::uint64_t>(width) * tokens > 0x7fffff00u || (seqs != 0 && width != 0 && table == nullptr)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    *out = Table{refs, blocks, tokens, table, nullptr, seqs, width, stride, (width + kRow - 1) / kRow};
    return static_cast<std::uint64_t>(seqs) * out->chunks > kMostWork ? HBFSIM_UNSUPPORTED : HBFSIM_OK;
}
bool tokens_ok(std::uint32_t n) { return n == 16 || n == 32 || n == 64 || n == 128; }

struct GrowSpace {
    std::size_t need, slot, found, writers, last, pair, bytes;
};
std::uint64_t slots_of(const Cache& c, std::uint32_t seqs, std::uint32_t tokens, bool offsets)
{
    return offsets ? tokens / c.tokens + std::uint64_t{2} * seqs : seqs;
}
GrowSpace grow_space(const Cache& c, std::uint32_t seqs, std::uint64_t slots)
{
    GrowSpace g{};
    std::size_t at = 0;
    const auto take = [&](std::size_t n) {
        const std::size_t here = at;
        at += up256(n);
        return here;
    };
    g.slot = take(slots * sizeof(int4));
    g.pair = take(seqs * sizeof(int2));
    g.need = take((slots + 1) * 4);
    g.found = take(slots * 4);
    g.writers = take(static_cast<std::size_t>(c.blocks) * 4);
    g.last = take(static_cast<std::size_t>(c.blocks) * 4);
    g.bytes = at;
    return g;
}

struct CompactSpace {
    std::uint32_t chunks;
    std::size_t count, moves, source, hole, bytes;
};
CompactSpace compact_space(const Cache& c)
{
    CompactSpace k{};
    k.chunks = (c.blocks + kChunk - 1) / kChunk;
    k.moves = 0;
    k.count = 256;
    k.source = k.count + up256(static_cast<std::size_t>(k.chunks) * 4);
    k.hole = k.source + up256((static_cast<std::size_t>(c.blocks) / 2 + 1) * 4);
    k.bytes = k.hole + up256((static_cast<std::size_t>(c.blocks) / 2 + 1) * 4);
    return k;
}

}  // namespace

#define HBF_API extern "C" __attribute__((visibility("default")))

HBF_API int hbfsim_amd_kv_copy_workspace(const hbfsim_amd_kv_cache* to, size_t n, size_t* bytes)
{
    Cache c{};
    const int rc = take_cache(to, &c);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    if (bytes == nullptr) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    *bytes = n == 0 ? 0 : static_cast<std::size_t>(c.blocks) * 4;
    return HBFSIM_OK;
}

HBF_API int hbfsim_amd_kv_copy(const hbfsim_amd_kv_cache* from, const hbfsim_amd_kv_cache* to, const int32_t* d_src,
                               const int32_t* d_dst, size_t n, void* d_workspace, size_t workspace_bytes, void* stream)
{
    Copy a{};
    int rc = take_cache(from, &a.from);
    if (rc == HBFSIM_OK) rc = take_cache(to, &a.to);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    a.same = same(a.from, a.to) ? 1 : 0;
    if (a.from.kv_heads != a.to.kv_heads || a.from.dim != a.to.dim || a.from.tokens != a.to.tokens ||
        (a.same == 0 && !apart(a.from, a.to))) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (n == 0) {
        return HBFSIM_OK;
    }
    if (d_src == nullptr || d_dst == nullptr || d_workspace == nullptr || !aligned16(d_workspace) ||
        workspace_bytes < static_cast<std::size_t>(a.to.blocks) * 4) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    a.p = piece_of(a.from);
    if (n > kMostWork / a.p.parts) {
        return HBFSIM_UNSUPPORTED;
    }
    a.src = d_src;
    a.dst = d_dst;
    a.n = static_cast<std::uint32_t>(n);
    a.owner = static_cast<std::int32_t*>(d_workspace);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 few((a.n + kThreads - 1) / kThreads);
    hipLaunchKernelGGL(k_kv_copy_clear, few, dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(k_kv_copy_claim, few, dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(k_kv_copy, dim3(a.n * a.p.parts), dim3(kThreads), 0, s, a);
    return checked(hipGetLastError());
}

HBF_API int hbfsim_amd_kv_hold(int32_t* d_refs, uint32_t blocks, const int32_t* d_table, uint32_t seqs, uint32_t width,
                               uint32_t stride, void* stream)
{
    Table t{};
    const int rc = take_table(d_refs, blocks, 1, const_cast<std::int32_t*>(d_table), seqs, width, stride, &t);
    if (rc != HBFSIM_OK || seqs == 0 || width == 0) {
        return rc;
    }
    hipLaunchKernelGGL(k_kv_hold, dim3(seqs * t.chunks), dim3(kThreads), 0, static_cast<hipStream_t>(stream), t);
    return checked(hipGetLastError());
}

HBF_API int hbfsim_amd_kv_release(int32_t* d_refs, uint32_t blocks, uint32_t block_tokens, int32_t* d_table,
                                  const int32_t* d_lens, uint32_t seqs, uint32_t width, uint32_t stride, void* stream)
{
    Table t{};
    if (!tokens_ok(block_tokens)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    const int rc = take_table(d_refs, blocks, block_tokens, d_table, seqs, width, stride, &t);
    if (rc != HBFSIM_OK || seqs == 0 || width == 0) {
        return rc;
    }
    t.lens = d_lens;
    hipLaunchKernelGGL(k_kv_release, dim3(seqs * t.chunks), dim3(kThreads), 0, static_cast<hipStream_t>(stream), t);
    return checked(hipGetLastError());
}

HBF_API int hbfsim_amd_kv_fork(int32_t* d_refs, uint32_t blocks, const int32_t* d_table, const int32_t* d_lens,
                               uint32_t seqs, uint32_t width, uint32_t stride, const int32_t* d_parents, uint32_t rows,
                               int32_t* d_out_table, int32_t* d_out_lens, void* stream)
{
    Fork a{};
    const int rc = take_table(d_refs, blocks, 1, const_cast<std::int32_t*>(d_table), seqs, width, stride, &a.t);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    const std::size_t out = static_cast<std::size_t>(rows) * width * 4, lens = static_cast<std::size_t>(rows) * 4;
    const std::size_t in = seqs == 0 ? 0 : ((static_cast<std::size_t>(seqs) - 1) * stride + width) * 4;
    if (rows > 0x7fffff00u || (rows != 0 && (d_parents == nullptr || d_out_lens == nullptr || (width != 0 && d_out_table == nullptr))) ||
        (rows != 0 && seqs != 0 && d_lens == nullptr) || meet(d_out_table, out, d_table, in) ||
        meet(d_out_table, out, d_refs, std::size_t{4} * blocks) || meet(d_out_table, out, d_parents, lens) ||
        meet(d_out_table, out, d_lens, std::size_t{4} * seqs) || meet(d_out_lens, lens, d_lens, std::size_t{4} * seqs) ||
        meet(d_out_lens, lens, d_parents, lens) || meet(d_out_lens, lens, d_table, in) || meet(d_out_table, out, d_out_lens, lens)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (a.t.chunks == 0) a.t.chunks = 1;  // lengths alone
    const std::uint64_t groups = (static_cast<std::uint64_t>(rows) + seqs) * a.t.chunks;
    if (groups > kMostWork) {
        return HBFSIM_UNSUPPORTED;
    }
    if (groups == 0) {
        return HBFSIM_OK;
    }
    a.t.lens = d_lens;
    a.parents = d_parents;
    a.rows = rows;
    a.out = d_out_table;
    a.out_lens = d_out_lens;
    hipLaunchKernelGGL(k_kv_fork, dim3(static_cast<std::uint32_t>(groups)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), a);
    return checked(hipGetLastError());
}

HBF_API int hbfsim_amd_kv_grow_workspace(const hbfsim_amd_kv_cache* cache, uint32_t seqs, uint32_t tokens, size_t* bytes)
{
    Cache c{};
    const int rc = take_cache(cache, &c);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    if (bytes == nullptr || seqs > 0x7fffff00u || tokens > 0x7fffff00u) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    *bytes = seqs == 0 ? 0 : grow_space(c, seqs, slots_of(c, seqs, tokens, true)).bytes;
    return HBFSIM_OK;
}

HBF_API int hbfsim_amd_kv_grow(const hbfsim_amd_kv_cache* cache, int32_t* d_refs, int32_t* d_table, const int32_t* d_lens,
                               const int32_t* d_first, uint32_t seqs, uint32_t tokens, uint32_t width, uint32_t stride,
                               int32_t* d_out_lens, int32_t* d_missing, void* d_workspace, size_t workspace_bytes,
                               void* stream)
{
    Grow a{};
    Table t{};
    int rc = take_cache(cache, &a.c);
    if (rc == HBFSIM_OK) rc = take_table(d_refs, a.c.blocks, a.c.tokens, d_table, seqs, width, stride, &t);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    if (tokens > 0x7fffff00u || (d_first == nullptr && tokens != seqs)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (seqs == 0) {
        return HBFSIM_OK;
    }
    const std::uint64_t slots = slots_of(a.c, seqs, tokens, d_first != nullptr);
    a.p = piece_of(a.c);
    if (slots > kMostGroups || static_cast<std::uint64_t>(seqs) * a.p.parts > kMostWork) {
        return HBFSIM_UNSUPPORTED;
    }
    const GrowSpace g = grow_space(a.c, seqs, slots);
    if (d_lens == nullptr || d_out_lens == nullptr || d_missing == nullptr || d_workspace == nullptr ||
        !aligned16(d_workspace) || workspace_bytes < g.bytes) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    a.refs = d_refs;
    a.table = d_table;
    a.lens = d_lens;
    a.first = d_first;
    a.seqs = seqs;
    a.tokens = tokens;
    a.width = width;
    a.stride = stride;
    a.slots = static_cast<std::uint32_t>(slots);
    a.out_lens = d_out_lens;
    a.missing = d_missing;
    unsigned char* ws = static_cast<unsigned char*>(d_workspace);
    a.slot = reinterpret_cast<int4*>(ws + g.slot);
    a.pair = reinterpret_cast<int2*>(ws + g.pair);
    a.need = reinterpret_cast<std::int32_t*>(ws + g.need);
    a.found = reinterpret_cast<std::int32_t*>(ws + g.found);
    a.writers = reinterpret_cast<std::int32_t*>(ws + g.writers);
    a.last = reinterpret_cast<std::int32_t*>(ws + g.last);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(k_kv_grow, dim3(1), dim3(kPlan), 0, s, a);
    hipLaunchKernelGGL(k_kv_grow_copy, dim3(seqs * a.p.parts), dim3(kThreads), 0, s, a);
    return checked(hipGetLastError());
}

HBF_API int hbfsim_amd_kv_compact_workspace(const hbfsim_amd_kv_cache* cache, size_t* bytes)
{
    Cache c{};
    const int rc = take_cache(cache, &c);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    if (bytes == nullptr) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    *bytes = compact_space(c).bytes;
    return HBFSIM_OK;
}

HBF_API int hbfsim_amd_kv_compact(const hbfsim_amd_kv_cache* cache, int32_t* d_refs, int32_t* d_table, uint32_t seqs,
                                  uint32_t width, uint32_t stride, int32_t* d_where, void* d_workspace,
                                  size_t workspace_bytes, void* stream)
{
    Compact a{};
    int rc = take_cache(cache, &a.c);
    if (rc == HBFSIM_OK) rc = take_table(d_refs, a.c.blocks, a.c.tokens, d_table, seqs, width, stride, &a.t);
    if (rc != HBFSIM_OK) {
        return rc;
    }
    const CompactSpace k = compact_space(a.c);
    if (d_where == nullptr || d_workspace == nullptr || !aligned16(d_workspace) || workspace_bytes < k.bytes) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    a.p = piece_of(a.c);
    const std::uint64_t items = std::uint64_t{a.c.blocks} / 2 * a.p.parts;
    const std::uint32_t movers = items < 4096 ? static_cast<std::uint32_t>(items) : 4096;
    const std::uint64_t groups = movers + static_cast<std::uint64_t>(seqs) * a.t.chunks;
    if (groups > kMostWork) {
        return HBFSIM_UNSUPPORTED;
    }
    a.where = d_where;
    a.chunks = k.chunks;
    unsigned char* ws = static_cast<unsigned char*>(d_workspace);
    a.moves = reinterpret_cast<std::uint32_t*>(ws + k.moves);
    a.count = reinterpret_cast<std::uint32_t*>(ws + k.count);
    a.source = reinterpret_cast<std::int32_t*>(ws + k.source);
    a.hole = reinterpret_cast<std::int32_t*>(ws + k.hole);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(k_kv_compact_count, dim3(k.chunks), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(k_kv_compact_plan, dim3(k.chunks), dim3(kThreads), 0, s, a);
    if (groups != 0) {
        hipLaunchKernelGGL(k_kv_compact, dim3(static_cast<std::uint32_t>(groups)), dim3(kThreads), 0, s, a, movers);
    }
    return checked(hipGetLastError());
}
