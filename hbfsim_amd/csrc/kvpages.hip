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

// One workgroup's part of a block, all of its loads before the first store.  A
// wave's 64 units are of one array, as a block's keys and values are whole KiB.
// Past the caches, as a block that moves is rarely read again soon: 8,003
// blocks of 35 KB (560 MB in and out) take 112 us, 5.0 TB/s, with non-temporal
// loads and stores, and a call 118, 121 with such stores alone, 124 with neither.
// (Measured on copies of a pool.  grow's few copies are read again in the same
// step and go the same way.)
constexpr int kUnits = 4;  // of a thread
__device__ inline void copy_part(const Cache& from, const Cache& to, const Piece& p, std::int32_t src, std::int32_t dst,
                                 std::uint32_t part)
{
    const std::uint32_t all = 2 * p.codes + p.bounds;
    const std::uint32_t end = (part + 1) * p.per < all ? (part + 1) * p.per : all;
    const std::size_t s = static_cast<std::size_t>(src), d = static_cast<std::size_t>(dst);
    const auto at = [&](const Cache& c, std::size_t id, std::uint32_t i) {
        return i < p.codes ? reinterpret_cast<u32x4*>(c.keys) + id * p.codes + i
               : i < 2 * p.codes ? reinterpret_cast<u32x4*>(c.values) + id * p.codes + (i - p.codes)
                                 : reinterpret_cast<u32x4*>(c.bounds) + id * p.bounds + (i - 2 * p.codes);
    };
    u32x4 x[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        const std::uint32_t i = part * p.per + k * kThreads + threadIdx.x;
        if (i < end) x[k] = __builtin_nontemporal_load(at(from, s, i));
    }
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        const std::uint32_t i = part * p.per + k * kThreads + threadIdx.x;
        if (i < end) __builtin_nontemporal_store(x[k], at(to, d, i));
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
constexpr std::uint32_t kFewPairs = 1024;

__device__ inline bool pair_at(const Copy& a, std::uint32_t i, std::int32_t* src, std::int32_t* dst)
{
    *src = a.src[i];
    *dst = a.dst[i];
    return inside(*src, a.from.blocks) && inside(*dst, a.to.blocks);
}
// Who copies to a block is settled in two launches before the copy, 4.7 and 4.6 us
// for 8,003 pairs; in one workgroup with a barrier they took 23, as one compute
// unit's atomics wait for one another.
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
// Pairs count only where both ids are of their pools.
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
// Every workgroup looks through the pairs itself: one launch instead of three.
// 4 pairs take 3.1 us against 6.2, 256 of 35 KB 5.3 against 8.8, 1,024 18.0
// against 20.7, 2,048 33.3 against 35.0; 4,096 take 75 against 64.  Every part of
// a block repeats the look, three of them here, 33 where a block has 0.5 MB, which
// is not measured: the border stays on the low side.
__global__ __launch_bounds__(kThreads) void k_kv_copy_few(Copy a)
{
    const std::uint32_t i = blockIdx.x / a.p.parts, part = blockIdx.x % a.p.parts;
    std::int32_t src, dst;
    const bool counts = pair_at(a, i, &src, &dst);
    bool taken = !counts;
    for (std::uint32_t j = threadIdx.x; j < a.n; j += kThreads) {
        std::int32_t s, d;
        if (pair_at(a, j, &s, &d)) taken |= (d == dst && j < i) || (a.same != 0 && d == src);
    }
    if (__syncthreads_or(taken) == 0) copy_part(a.from, a.to, a.p, src, dst, part);
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

// Tables are walked by workgroups of 1,024 entries.  Bound by the launch, and for
// large tables by the atomics: hold takes 2.7 us for 8 rows of 512 entries, 6.5 for
// 64 of 2,048 and 20.7 for 256 of them where every entry names another block, and
// 131 for 64 of 2,048 that name 100 blocks (1,300 atomics on one address);
// release 6.7 for 256 rows of 193,000 entries, of which 65,000 leave, and 3.1 for 64
// rows of which few do.
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
    bool net;
};
// The first rows * chunks workgroups write the new rows, the others change the
// old rows' counts: by their children less one, which each finds among the
// parents, or by one down where the new rows count one up themselves.  64 rows
// of up to 2,048 entries continued by 256 take 6.5 us, 8 rows 3.0.
__global__ __launch_bounds__(kThreads) void k_kv_fork(Fork a)
{
    const std::uint32_t r = blockIdx.x / a.t.chunks, chunk = blockIdx.x % a.t.chunks;
    if (r < a.rows) {
        const std::int32_t p = a.parents[r];
        const bool there = inside(p, a.t.seqs);
        const std::int32_t* row = a.t.table + static_cast<std::size_t>(there ? p : 0) * a.t.stride;
        each_entry(a.t, chunk, [&](std::uint32_t i) {
            const std::int32_t id = there ? row[i] : -1;
            a.out[static_cast<std::size_t>(r) * a.t.width + i] = id;
            if (!a.net && inside(id, a.t.blocks)) atomicAdd(&a.t.refs[id], 1);
        });
        if (chunk == 0 && threadIdx.x == 0) a.out_lens[r] = there ? a.t.lens[p] : 0;
        return;
    }
    const std::uint32_t s = r - a.rows;
    __shared__ std::int32_t s_count[kThreads / kWave];
    std::int32_t children = 0;
    if (a.net) {
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
    std::uint32_t vector;  // counts may be loaded 16 bytes at a time
    std::int32_t* out_lens;
    std::int32_t* missing;
    // workspace
    std::int32_t* need;     // [slots + 1]: new blocks of the slots before
    int4* slot;             // [slots]: sequence, place, the row's block or what to do without
    std::int32_t* found;    // [slots]: free blocks, ascending
    std::int32_t* writers;  // [blocks]: slots that write to a shared block, and the last of them
    std::int32_t* last;
    int2* pair;             // [seqs]: content to copy, source and destination
    std::int32_t* count;    // [tiles] of the pool: free blocks; or null
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
// Atomics' results as they are now.
__device__ inline std::int32_t now(const std::int32_t* p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
    __syncthreads();
    return total;
}

// Bits of a thread's 8 blocks from id0 on that are free.
__device__ inline std::uint32_t free_of_8(const Grow& a, std::uint64_t id0)
{
    std::int32_t r[8];
    if (a.vector != 0 && id0 + 8 <= a.c.blocks) {
        *reinterpret_cast<int4*>(r) = *reinterpret_cast<const int4*>(a.refs + id0);
        *reinterpret_cast<int4*>(r + 4) = *reinterpret_cast<const int4*>(a.refs + id0 + 4);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) r[k] = id0 + k < a.c.blocks ? a.refs[id0 + k] : 1;
    }
    std::uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) bits |= r[k] <= 0 ? 1u << k : 0u;
    return bits;
}
// Sums of numbers below 2^kBits before each thread's, and of all.
template <int kBits>
__device__ inline std::int32_t before_small(std::uint32_t x, std::int32_t* all)
{
    __shared__ std::int32_t s_wave[kPlanWaves];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const unsigned long long below = (1ull << lane) - 1;
    std::int32_t mine = 0, sum = 0;
#pragma unroll
    for (int b = 0; b < kBits; ++b) {
        const unsigned long long votes = __ballot((x >> b & 1u) != 0);
        mine += __popcll(votes & below) << b;
        sum += __popcll(votes) << b;
    }
    __syncthreads();
    if (lane == 0) s_wave[wave] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int i = 0; i < kPlanWaves; ++i) {
        mine += i < wave ? s_wave[i] : 0;
        sum += s_wave[i];
    }
    *all = sum;
    return mine;
}

// Free blocks of every tile, a workgroup each: for pools that one compute unit
// would look through for longer than a launch takes.
constexpr std::uint32_t kTile = 8 * kPlan;  // blocks
__global__ __launch_bounds__(kPlan) void k_kv_grow_count(Grow a)
{
    std::int32_t all;
    before_small<4>(__popc(free_of_8(a, std::uint64_t{blockIdx.x} * kTile + std::uint64_t{8} * threadIdx.x)), &all);
    if (threadIdx.x == 0) a.count[blockIdx.x] = all;
}

// The first `want` free blocks, in order, to put(rank, id); returns how many
// there are, all of them where they are fewer.  `tile` holds a thread's of the
// first tile, and each tile is on its way while the one before is counted; with
// counts, tiles without a free block are left out.
// A compute unit reads 33 GB/s so, a tile in 1.03 us: a step of 64 sequences
// takes 6 us where the first tile has their blocks, and without counts 15 where
// the first half of 131,072 blocks is in use, 22 where nearly all are; with
// them 10 wherever the free ones lie, also of 500,000 (70 without).
template <typename F>
__device__ inline std::int32_t first_free(const Grow& a, std::uint32_t tile, std::int32_t want, F put)
{
    __shared__ int2 s_tile[kPlan];  // index, free blocks before it
    const auto take = [&](std::uint32_t bits, std::int32_t rank, std::uint64_t id0) {
        for (; bits != 0 && rank < want; bits &= bits - 1) put(rank++, static_cast<std::int32_t>(id0) + __ffs(bits) - 1);
    };
    const std::uint64_t mine = std::uint64_t{8} * threadIdx.x;
    std::int32_t free = 0, all;
    if (a.count == nullptr) {
        for (std::uint64_t from = 0; free < want && from < a.c.blocks; from += kTile) {
            const std::uint32_t next = from + kTile < a.c.blocks ? free_of_8(a, from + kTile + mine) : 0;
            const std::int32_t rank = free + before_small<4>(__popc(tile), &all);
            take(tile, rank, from + mine);
            free += all;
            tile = next;
        }
        return free;
    }
    const std::uint32_t tiles = (a.c.blocks + kTile - 1) / kTile;
    for (std::uint32_t group = 0; free < want && group < tiles; group += kPlan) {
        const std::int32_t count = group + threadIdx.x < tiles ? a.count[group + threadIdx.x] : 0;
        std::int32_t used;
        const std::int32_t rank = free + before(count, &all);
        const bool use = count > 0 && rank < want;
        const std::int32_t at = before_small<1>(use ? 1 : 0, &used);
        if (use) s_tile[at] = int2{static_cast<int>(group + threadIdx.x), rank};
        __syncthreads();
        const auto from = [&](int i) { return static_cast<std::uint64_t>(s_tile[i].x) * kTile + mine; };
        std::uint32_t bits = used > 0 ? free_of_8(a, from(0)) : 0;
        for (int i = 0; i < used; ++i) {
            const std::uint32_t next = i + 1 < used ? free_of_8(a, from(i + 1)) : 0;
            std::int32_t here;
            const std::int32_t first = before_small<4>(__popc(bits), &here);
            take(bits, s_tile[i].y + first, from(i));
            bits = next;
        }
        __syncthreads();
        free += all;
    }
    return free;
}

// One workgroup plans: what each slot writes to, who keeps a shared block, how
// many blocks are wanted, the first free ones, who gets them.  A slot is a block
// that a sequence may write to, as in append.  Every step needs the one before
// of all slots, so it is a chain of trips to memory and barriers, no work to
// spread: 11.4 us for 17 chunks of 35,769 tokens (1,151 slots), 25 for 4,000
// sequences of one token.  Slots go through global memory between the barriers;
// a few a thread would fit the LDS as well, as one does below.
__global__ __launch_bounds__(kPlan) void k_kv_grow(Grow a)
{
    constexpr std::uint32_t kHeld = 4096;  // sequences whose parts lie in LDS
    __shared__ std::int32_t s_base[kHeld + 1];
    __shared__ int2 s_part[kHeld];
    const std::uint32_t t = a.c.tokens;
    const bool held = a.seqs <= kHeld;
    for (std::uint32_t s = threadIdx.x; s < a.seqs; s += kPlan) {
        a.pair[s] = int2{-1, -1};
        if (held) {
            const Part part = part_of(a, s);
            s_part[s] = int2{static_cast<int>(part.from), static_cast<int>(part.to)};
            s_base[s] = static_cast<std::int32_t>(base_of(a, s));
        }
    }
    if (held && threadIdx.x == 0) s_base[a.seqs] = static_cast<std::int32_t>(a.slots);
    std::uint32_t tile = free_of_8(a, std::uint64_t{8} * threadIdx.x);
    __syncthreads();
    const auto base = [&](std::uint32_t s) {
        return held ? static_cast<std::uint32_t>(s_base[s]) : s < a.seqs ? base_of(a, s) : a.slots;
    };
    const auto parts = [&](std::uint32_t s) { return held ? Part{s_part[s].x, s_part[s].y} : part_of(a, s); };
    bool shared = false;
    for (std::uint32_t i = threadIdx.x; i < a.slots; i += kPlan) {
        std::uint32_t s = i;
        if (a.first != nullptr) {
            std::uint32_t lo = 0, hi = a.seqs;  // the last sequence whose slots begin at or before i
            while (hi - lo > 1) {
                const std::uint32_t mid = lo + (hi - lo) / 2;
                if (base(mid) <= i) lo = mid; else hi = mid;
            }
            s = lo;
        }
        int4 slot = {static_cast<int>(s), 0, kIdle, 0};
        const Part part = parts(s);
        const std::int64_t place = part.from / t + (static_cast<std::int64_t>(i) - base(s));
        if (i >= base(s) && place * t < part.to && (part.to - 1) / t < static_cast<std::int64_t>(a.width)) {
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
    if (__syncthreads_or(shared)) {
        for (std::uint32_t i = threadIdx.x; i < a.slots; i += kPlan) {
            const int4 slot = a.slot[i];
            if (slot.z >= 0 && slot.w > 1) {
                atomicAdd(&a.writers[slot.z], 1);
                atomicMax(&a.last[slot.z], static_cast<std::int32_t>(i));
            }
        }
        __syncthreads();
    }
    const auto fresh = [&](std::uint32_t i) {
        const int4 slot = a.slot[i];
        if (slot.z < 0 || slot.w <= 1) return slot.z == kNew;
        return now(&a.writers[slot.z]) < slot.w || now(&a.last[slot.z]) != static_cast<std::int32_t>(i);
    };
    const auto fresh_alone = [&](std::uint32_t i) {  // no shared block is kept
        const int4 slot = a.slot[i];
        return slot.z == kNew || (slot.z >= 0 && slot.w > 1);
    };
    std::int32_t want = count_needs(a, fresh);
    const std::int32_t free = first_free(a, tile, want, [&](std::int32_t rank, std::int32_t id) { a.found[rank] = id; });
    const bool enough = free >= want;
    if (!enough) want = count_needs(a, fresh_alone);
    __syncthreads();
    const auto granted = [&](std::uint32_t s, const Part& part) {
        if (part.to > 0 && (part.to - 1) / t >= static_cast<std::int64_t>(a.width)) return false;
        const std::int32_t from = a.need[base(s)], to = a.need[base(s + 1)];
        return enough || to == from || to <= free;
    };
    for (std::uint32_t i = threadIdx.x; i < a.slots; i += kPlan) {
        const int4 slot = a.slot[i];
        if (slot.z == kIdle) continue;
        const Part part = parts(slot.x);
        const bool gets = enough ? fresh(i) : fresh_alone(i);
        if ((!gets && slot.z != kStale) || !granted(slot.x, part)) continue;
        std::int32_t* entry = a.table + static_cast<std::size_t>(slot.x) * a.stride + slot.y;
        if (!gets) {
            *entry = -1;
            continue;
        }
        const std::int32_t id = a.found[a.need[i]];
        *entry = id;
        a.refs[id] = 1;
        if (slot.z >= 0) {
            atomicSub(&a.refs[slot.z], 1);
            if (static_cast<std::int64_t>(slot.y) * t < part.from) a.pair[slot.x] = int2{slot.z, id};
        }
    }
    __syncthreads();  // the lengths may become the new ones
    for (std::uint32_t s = threadIdx.x; s < a.seqs; s += kPlan) {
        const Part part = parts(s);
        std::int32_t lacks = 0;
        if (!granted(s, part)) {
            const std::int64_t from = part.from / t, to = (part.to - 1) / t + 1, width = a.width;
            lacks = to > width ? static_cast<std::int32_t>(to - (from > width ? from : width))
                               : a.need[base(s + 1)] - a.need[base(s)];
        }
        a.missing[s] = lacks;
        a.out_lens[s] = lacks != 0 ? 0 : a.lens[s];
    }
}

// The same for at most kPlan slots, a thread each: what the slots share lies in
// LDS, and the first free blocks are looked for while the rows come in: 5.4 us
// for 64 sequences of one token, a microsecond more for 1,024; the form above
// takes five more for 1,500.
constexpr int kShared = 2 * kPlan;  // of the table of shared blocks

__global__ __launch_bounds__(kPlan) void k_kv_grow_few(Grow a)
{
    __shared__ std::int32_t s_base[kPlan + 1], s_need[kPlan + 1], s_found[kPlan];
    __shared__ int2 s_part[kPlan], s_pair[kPlan];
    __shared__ std::int32_t s_id[kShared], s_writers[kShared], s_last[kShared];
    const int i = threadIdx.x;
    const std::int64_t width = a.width;
    const std::uint32_t shift = 4 + a.c.tile_shift;
    std::int32_t len = 0;
    Part own{0, 0};
    if (i < static_cast<int>(a.seqs)) {
        len = a.lens[i];
        own = part_of(a, i);
        s_part[i] = int2{static_cast<int>(own.from), static_cast<int>(own.to)};
        s_base[i] = static_cast<std::int32_t>(base_of(a, i));
        s_pair[i] = int2{-1, -1};
    }
    if (i == 0) s_base[a.seqs] = static_cast<std::int32_t>(a.slots);
#pragma unroll
    for (int k = 0; k < kShared; k += kPlan) {
        s_id[k + i] = -1;
        s_writers[k + i] = 0;
        s_last[k + i] = -1;
    }
    std::uint32_t tile = free_of_8(a, std::uint64_t{8} * i);
    __syncthreads();
    std::uint32_t s = i;
    int z = kIdle;
    std::int32_t refs = 0;
    std::int64_t place = 0;
    bool begun = false;
    if (i < static_cast<int>(a.slots)) {
        if (a.first != nullptr) {
            std::uint32_t lo = 0, hi = a.seqs;
            while (hi - lo > 1) {
                const std::uint32_t mid = lo + (hi - lo) / 2;
                if (s_base[mid] <= i) lo = mid; else hi = mid;
            }
            s = lo;
        }
        const int2 part = s_part[s];
        place = (part.x >> shift) + static_cast<std::int64_t>(i - s_base[s]);
        if (i >= s_base[s] && place << shift < part.y && (part.y - 1) >> shift < width) {
            const std::int32_t id = a.table[static_cast<std::size_t>(s) * a.stride + place];
            const bool named = inside(id, a.c.blocks);
            refs = named ? a.refs[id] : 0;
            begun = place << shift < part.x;
            z = refs > 0 ? id : !begun ? kNew : named ? kStale : kIdle;
        }
    }
    const bool shared = z >= 0 && refs > 1;
    bool keeps = !shared;
    if (__syncthreads_or(shared)) {
        std::uint32_t h = 0;
        if (shared) {
            h = static_cast<std::uint32_t>(z) * 2654435761u >> 21;
            for (;;) {  // at most half of the places are taken
                const std::int32_t was = atomicCAS(&s_id[h], -1, z);
                if (was == -1 || was == z) break;
                h = (h + 1) % kShared;
            }
            atomicAdd(&s_writers[h], 1);
            atomicMax(&s_last[h], i);
        }
        __syncthreads();
        if (shared) keeps = s_writers[h] >= refs && s_last[h] == i;
    }
    bool fresh = z == kNew || (z >= 0 && !keeps);
    std::int32_t want;
    std::int32_t at = before_small<1>(fresh ? 1 : 0, &want);
    const std::int32_t free = first_free(a, tile, want, [&](std::int32_t rank, std::int32_t id) { s_found[rank] = id; });
    const bool enough = free >= want;
    if (!enough) {  // no shared block is kept
        fresh = z == kNew || shared;
        at = before_small<1>(fresh ? 1 : 0, &want);
    }
    s_need[i] = at;
    if (i == 0) s_need[kPlan] = want;
    __syncthreads();
    const auto needs = [&](std::uint32_t q) { return int2{s_need[s_base[q]], s_need[s_base[q + 1]]}; };
    const auto granted = [&](std::uint32_t q, const int2& part) {
        const int2 need = needs(q);
        return !(part.y > 0 && (part.y - 1) >> shift >= width) && (enough || need.x == need.y || need.y <= free);
    };
    if ((fresh || z == kStale) && granted(s, s_part[s])) {
        std::int32_t* entry = a.table + static_cast<std::size_t>(s) * a.stride + place;
        if (!fresh) {
            *entry = -1;
        } else {
            const std::int32_t id = s_found[at];
            *entry = id;
            a.refs[id] = 1;
            if (z >= 0) {
                atomicSub(&a.refs[z], 1);
                if (begun) s_pair[s] = int2{z, id};
            }
        }
    }
    __syncthreads();
    if (i < static_cast<int>(a.seqs)) {
        std::int32_t lacks = 0;
        if (!granted(i, s_part[i])) {
            const std::int64_t from = own.from >> shift, to = ((own.to - 1) >> shift) + 1;
            const int2 need = needs(i);
            lacks = to > width ? static_cast<std::int32_t>(to - (from > width ? from : width)) : need.y - need.x;
        }
        a.missing[i] = lacks;
        a.out_lens[i] = lacks != 0 ? 0 : len;
        a.pair[i] = s_pair[i];
    }
}

// The planned copies, at most kCopiers workgroups for all sequences' parts, as
// most steps have few; 3.2 us for 64 sequences of which a third part with a
// block, 2.0 where none does.  For 4,000 sequences and blocks of 34 parts a
// workgroup each cost 4 us more of such a step, and where all are copied (0.53
// GB of blocks of 128 tokens for 1,000) 93 us against 98.
constexpr std::uint32_t kCopiers = 8192;
__global__ __launch_bounds__(kThreads) void k_kv_grow_copy(Grow a)
{
    for (std::uint32_t i = blockIdx.x; i < a.seqs * a.p.parts; i += gridDim.x) {
        const int2 pair = a.pair[i / a.p.parts];
        if (pair.x >= 0) copy_part(a.c, a.c, a.p, pair.x, pair.y, i % a.p.parts);
    }
}

// ---- compact ------------------------------------------------------------------

constexpr std::uint32_t kChunk = kThreads * 4;  // blocks of a workgroup

struct Compact {
    Cache c;
    Piece p;
    Table t;
    std::int32_t* where;
    std::uint32_t chunks;
    std::uint32_t vector;  // counts and `where` may be moved 16 bytes at a time
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

// The plan in two launches: blocks in use of each 1,024, then every workgroup
// sums those before its own.  4.5 and 4.8 us for 42,000 blocks.
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

// Both steps in one workgroup, for pools of up to kFewBlocks: a wave takes a run
// of them, 256 at a time, and keeps which are in use as bits.
// (4,000 blocks: 10.1 us against 13.1 in two launches; 8,000: 12.1 and 13.4;
// 16,000: 14.8 and 14.2, and 65,000: 32.8 and 19.5.)
constexpr int kRounds = 2;
constexpr std::uint32_t kFewBlocks = kPlanWaves * kRounds * 256;

__global__ __launch_bounds__(kPlan) void k_kv_compact_plan_one(Compact a)
{
    __shared__ std::uint32_t s_live[kPlanWaves], s_front[kPlanWaves];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const std::uint32_t run = (a.c.blocks + kPlanWaves * 256 - 1) / (kPlanWaves * 256) * 256;
    const std::uint32_t first = wave * run + lane * 4;
    std::uint32_t used = 0;
#pragma unroll
    for (int n = 0; n < kRounds; ++n) {
        const std::uint32_t id = first + n * 256;
        if (n * 256 < static_cast<int>(run)) {
            std::int32_t r[4] = {0, 0, 0, 0};
            if (a.vector != 0 && id + 4 <= a.c.blocks) {
                *reinterpret_cast<int4*>(r) = *reinterpret_cast<const int4*>(a.t.refs + id);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) r[k] = id + k < a.c.blocks ? a.t.refs[id + k] : 0;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) used |= r[k] > 0 ? 1u << (4 * n + k) : 0u;
        }
    }
    const auto wave_total = [&](std::uint32_t x) {
#pragma unroll
        for (int k = 1; k < kWave; k *= 2) x += __shfl_xor(x, k);
        return x;
    };
    const std::uint32_t mine = wave_total(__popc(used));
    if (lane == 0) s_live[wave] = mine;
    __syncthreads();
    std::uint32_t at = 0, live = 0;
#pragma unroll
    for (int i = 0; i < kPlanWaves; ++i) {
        at += i < wave ? s_live[i] : 0;
        live += s_live[i];
    }
    std::uint32_t front = 0;  // blocks in use before the front's end
#pragma unroll
    for (int n = 0; n < kRounds; ++n) {
        const std::uint32_t id = first + n * 256;
        const std::uint32_t ahead = id >= live ? 0 : live - id < 4 ? live - id : 4;
        front += __popc(used >> (4 * n) & ((1u << ahead) - 1));
    }
    front = wave_total(front);
    if (lane == 0) s_front[wave] = front;
    __syncthreads();
    front = 0;
#pragma unroll
    for (int i = 0; i < kPlanWaves; ++i) front += s_front[i];
    const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
    for (std::uint32_t n = 0; n < kRounds; ++n) {
        if (n * 256 >= run) break;
        const std::uint32_t id0 = first + n * 256, four = used >> (4 * n) & 15u;
        std::uint32_t rank = at;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned long long votes = __ballot((four >> k & 1u) != 0);
            rank += __popcll(votes & below);
            at += __popcll(votes);
        }
        std::int32_t to[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const std::uint32_t id = id0 + k;
            to[k] = -1;
            if ((four >> k & 1u) != 0) {
                to[k] = static_cast<std::int32_t>(id);
                if (id >= live) {
                    a.source[rank - front] = static_cast<std::int32_t>(id);
                    to[k] = kMoves - static_cast<std::int32_t>(rank - front);
                }
                ++rank;
            } else if (id < live) {
                a.hole[id - rank] = static_cast<std::int32_t>(id);
            }
        }
        if (a.vector != 0 && id0 + 4 <= a.c.blocks) {
            *reinterpret_cast<int4*>(a.where + id0) = *reinterpret_cast<const int4*>(to);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (id0 + k < a.c.blocks) a.where[id0 + k] = to[k];
            }
        }
    }
    if (threadIdx.x == 0) *a.moves = live - front;
}

// The first workgroups move blocks, those from `movers` on the table's entries.
// An entry's block may get its place in `where` meanwhile: either form says it.
// 7,070 blocks of 35 KB (495 MB in and out) take 94 us, 5.3 TB/s.
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
    p.parts = (all + kUnits * kThreads - 1) / (kUnits * kThreads);
    p.per = ((all + p.parts - 1) / p.parts + kWave - 1) / kWave * kWave;
    return p;
}

std::size_t copy_bytes(const Cache& to, std::size_t n) { return n <= kFewPairs ? 0 : static_cast<std::size_t>(to.blocks) * 4; }
std::size_t block_bytes(const Cache& c) { return static_cast<std::size_t>(c.kv_heads) * c.tokens * c.dims; }

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
    std::size_t need, slot, found, writers, last, pair, count, bytes;
};
std::uint64_t slots_of(const Cache& c, std::uint32_t seqs, std::uint32_t tokens, bool offsets)
{
    return offsets ? tokens / c.tokens + std::uint64_t{2} * seqs : seqs;
}
// Blocks up to which the planning workgroup looks for free ones without counts,
// which cost 3.5 us: a step of 64 sequences in a pool of 60,000 takes 6 us where
// the first tile has their blocks, 12 where only the last ones do, as in a pool
// that hands out the lowest and is nearly full, and with counts 9.5 wherever they
// lie.  (From about 28,000 blocks on counts are the shorter way to the last ones.)
constexpr std::uint32_t kScanned = 65536;
// Where a thread takes a slot, the plan lies in LDS and only the pairs in memory.
GrowSpace grow_space(const Cache& c, std::uint32_t seqs, std::uint64_t slots)
{
    GrowSpace g{};
    std::size_t at = 0;
    const auto take = [&](std::size_t n) {
        const std::size_t here = at;
        at += up256(n);
        return here;
    };
    g.pair = take(seqs * sizeof(int2));
    if (c.blocks > kScanned) g.count = take((static_cast<std::size_t>(c.blocks) + kTile - 1) / kTile * 4);
    if (slots > kPlan) {
        g.slot = take(slots * sizeof(int4));
        g.need = take((slots + 1) * 4);
        g.found = take(slots * 4);
        g.writers = take(static_cast<std::size_t>(c.blocks) * 4);
        g.last = take(static_cast<std::size_t>(c.blocks) * 4);
    }
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
    *bytes = copy_bytes(c, n);
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
    const std::size_t need = copy_bytes(a.to, n);
    if (d_src == nullptr || d_dst == nullptr || workspace_bytes < need ||
        (need != 0 && (d_workspace == nullptr || !aligned16(d_workspace)))) {
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
    const dim3 every(a.n * a.p.parts);
    if (a.n <= kFewPairs) {
        hipLaunchKernelGGL(k_kv_copy_few, every, dim3(kThreads), 0, s, a);
    } else {
        const dim3 pairs((a.n + kThreads - 1) / kThreads);
        hipLaunchKernelGGL(k_kv_copy_clear, pairs, dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL(k_kv_copy_claim, pairs, dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL(k_kv_copy, every, dim3(kThreads), 0, s, a);
    }
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
    if (rows > 0x7fffff00u ||
        (rows != 0 && (d_parents == nullptr || d_out_lens == nullptr || (width != 0 && d_out_table == nullptr))) ||
        (rows != 0 && seqs != 0 && d_lens == nullptr) || meet(d_out_table, out, d_table, in) ||
        meet(d_out_table, out, d_refs, std::size_t{4} * blocks) || meet(d_out_table, out, d_parents, lens) ||
        meet(d_out_table, out, d_lens, std::size_t{4} * seqs) || meet(d_out_lens, lens, d_lens, std::size_t{4} * seqs) ||
        meet(d_out_lens, lens, d_parents, lens) || meet(d_out_lens, lens, d_table, in) ||
        meet(d_out_lens, lens, d_refs, std::size_t{4} * blocks) || meet(d_out_table, out, d_out_lens, lens)) {
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
    // Children are looked for among all rows in each old row's workgroups; counts
    // of their own cost each entry two atomics instead.  1,024 rows of 2,048
    // entries: 57 us against 160, 16,384 of 256: 134 and 315, of 16: 88 and 24,
    // 1,024 of 16: 5.7 and 5.5.
    a.net = rows <= 1024 || rows <= std::uint64_t{128} * width;
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
    a.vector = aligned16(d_refs) ? 1 : 0;
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
    if (a.c.blocks > kScanned) {
        a.count = reinterpret_cast<std::int32_t*>(ws + g.count);
        hipLaunchKernelGGL(k_kv_grow_count, dim3((a.c.blocks + kTile - 1) / kTile), dim3(kPlan), 0, s, a);
    }
    if (a.slots <= kPlan) {
        hipLaunchKernelGGL(k_kv_grow_few, dim3(1), dim3(kPlan), 0, s, a);
    } else {
        hipLaunchKernelGGL(k_kv_grow, dim3(1), dim3(kPlan), 0, s, a);
    }
    const std::uint32_t parts = seqs * a.p.parts;
    hipLaunchKernelGGL(k_kv_grow_copy, dim3(parts < kCopiers ? parts : kCopiers), dim3(kThreads), 0, s, a);
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
    a.vector = aligned16(d_refs) && aligned16(d_where) ? 1 : 0;
    a.chunks = k.chunks;
    unsigned char* ws = static_cast<unsigned char*>(d_workspace);
    a.moves = reinterpret_cast<std::uint32_t*>(ws + k.moves);
    a.count = reinterpret_cast<std::uint32_t*>(ws + k.count);
    a.source = reinterpret_cast<std::int32_t*>(ws + k.source);
    a.hole = reinterpret_cast<std::int32_t*>(ws + k.hole);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.c.blocks <= kFewBlocks) {
        hipLaunchKernelGGL(k_kv_compact_plan_one, dim3(1), dim3(kPlan), 0, s, a);
    } else {
        hipLaunchKernelGGL(k_kv_compact_count, dim3(k.chunks), dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL(k_kv_compact_plan, dim3(k.chunks), dim3(kThreads), 0, s, a);
    }
    if (groups != 0) {
        hipLaunchKernelGGL(k_kv_compact, dim3(static_cast<std::uint32_t>(groups)), dim3(kThreads), 0, s, a, movers);
    }
    return checked(hipGetLastError());
}
