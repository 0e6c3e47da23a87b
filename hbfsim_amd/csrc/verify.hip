// verify.hip -- which of a step's drafted tokens stay, and the token behind
// them, from the target's and the draft's probabilities and given random
// numbers.
//
// No counterpart in the reference.  Draft x after row r stays while
//   u[r] q_r(x) < p_r(x),
// a product of two 24-bit numbers, exact in 64 bits.  At the first row where it
// does not, the next token is drawn from max(p - q, 0), so that what a sequence
// gains is distributed as the target alone would have it; behind the last draft
// it is drawn from p.  Probabilities become whole numbers P = 2^40 p (f32 holds
// 24 bits, so a p above 2^-17 keeps all of them; below that a weight is off by
// at most 2^-41, one of p - q by 2^-40, and the sum by as much times the
// vocabulary: the price of sums that do not depend on their order) and are
// summed in 64 bits: vocabularies up to 2^22 fit.  What draws is a float: one of
// 24 bits tells 2^-24 of the sum apart.
//
// Bound by memory where rows are long: one row of p a sequence, and one of q
// where a draft was refused, are read; of the other rows one element each.
#include "kvcache.hpp"

namespace {

using namespace hbfamd::kv;

constexpr int kThreads = 256;

typedef unsigned long long u64;

// What the second launch needs of a sequence, so that it need not look it up.
struct alignas(16) State {
    int4 drafts;                // accepted, whether a draft was refused, that draft
    std::int32_t begin, count;  // its rows
    float uniform;              // of the last one
};

struct Verify {
    const void* target;
    const void* draft;  // or null
    std::int64_t target_stride, draft_stride;
    const std::int32_t* tokens;
    const float* uniform;
    const std::int32_t* first;
    const std::int32_t* lens;
    const std::int32_t* stored;  // lengths before the step, or null
    std::uint32_t seqs, rows, vocab, regions;
    std::uint32_t vector;  // rows of both may be loaded 16 bytes at a time
    std::int32_t* out;
    std::int32_t* gained;
    std::int32_t* out_lens;
    State* state;  // [seqs]
    u64* sums;     // [seqs][regions]: of what is drawn from
};

// A length below the sequence's rows says that the step left it out.
// It is asked for where a sequence's results are at hand: a wait for it before
// the rows are read costs 64 sequences over 151,936 tokens 0.4 us.
__device__ inline std::int32_t length_of(const Verify& a, std::uint32_t s)
{
    return a.lens == nullptr ? 0x7fffffff : a.lens[s];
}
// A sequence's rows, none if they do not describe the batch.
struct Rows {
    std::int64_t begin;
    std::int32_t count;
};
__device__ inline Rows rows_of(const Verify& a, std::uint32_t s)
{
    std::int64_t begin = s, count = 1;
    if (a.first != nullptr) {
        begin = a.first[s];
        count = a.first[s + 1] - begin;
    }
    if (begin < 0 || count <= 0 || begin + count > a.rows) {
        return Rows{begin, 0};
    }
    return Rows{begin, static_cast<std::int32_t>(count)};
}

__device__ inline float share(float x) { return fminf(fmaxf(x, 0.0f), 1.0f); }
// rint(2^40 x) = 2^20 a + b in 32-bit arithmetic: 2^20 x has 24 bits, so its
// whole part a and its fraction are exact, and one fused step rounds 2^20 of
// the fraction to a whole number above 2^23 (to even: 2^20 a is even).  Five
// instructions of full rate, where 64-bit floats took one workgroup 13.4 us for
// two rows of 32,000.
struct Parts {
    std::int32_t a, b;
};
__device__ inline Parts parts_of(float x)
{
    const float t = x * 0x1p20f;
    const float b = __builtin_fmaf(__builtin_amdgcn_fractf(t), 0x1p20f, 0x1p23f);
    return Parts{static_cast<std::int32_t>(t), static_cast<std::int32_t>(__float_as_uint(b) - 0x4b000000u)};
}
__device__ inline u64 joined(const Parts& x) { return static_cast<u64>((static_cast<std::int64_t>(x.a) << 20) + x.b); }

// A wave's part of a row: kSteps consecutive KiB, 16 bytes a lane each, zeros
// past the row's end.
template <typename T, int kSteps>
__device__ inline void load_region(const T* row, std::uint32_t region, std::uint32_t vocab, bool vector, u32x4 (&x)[kSteps])
{
    constexpr int kEach = 16 / sizeof(T);
    const std::uint32_t from = region * kSteps * kWave * kEach, mine = from + threadIdx.x % kWave * kEach;
    if (vector && from + kSteps * kWave * kEach <= vocab) {  // all of the loads at once
#pragma unroll
        for (int i = 0; i < kSteps; ++i) x[i] = *reinterpret_cast<const u32x4*>(row + mine + i * kWave * kEach);
        return;
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const std::uint32_t e = mine + i * kWave * kEach;
        union {
            u32x4 v;
            T t[kEach];
        } u;
        u.v = u32x4{0u, 0u, 0u, 0u};
        if (vector && e + kEach <= vocab) {
            u.v = *reinterpret_cast<const u32x4*>(row + e);
        } else {
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                if (e + k < vocab) u.t[k] = row[e + k];
            }
        }
        x[i] = u.v;
    }
}

// What the next token is drawn from: P where no draft was refused, otherwise
// max(P - Q, 0), or P but for the refused token.
enum class From { kTarget, kRest, kOthers };
__device__ inline From from_of(const Verify& a, const int4& state)
{
    return state.y == 0 ? From::kTarget : a.draft != nullptr ? From::kRest : From::kOthers;
}

template <typename T, int kSteps>
struct Region {
    static constexpr int kEach = 16 / sizeof(T);
    u32x4 p[kSteps], q[kSteps];  // q only where the draft's row is taken off
    std::uint32_t mine;          // index of the lane's first element

    __device__ inline void load(const Verify& a, std::int64_t row, From from, std::uint32_t region)
    {
        mine = region * kSteps * kWave * kEach + threadIdx.x % kWave * kEach;
        load_region<T, kSteps>(static_cast<const T*>(a.target) + row * a.target_stride, region, a.vocab, a.vector != 0, p);
        if (from == From::kRest) {
            load_region<T, kSteps>(static_cast<const T*>(a.draft) + row * a.draft_stride, region, a.vocab, a.vector != 0, q);
        }
    }
    // Element j of step i, without token `out`.  Where q is not below p, neither
    // is its whole number.
    __device__ inline Parts weight(int i, int j, From from, std::uint32_t out) const
    {
        const float x = element(p[i], j);
        Parts w = parts_of(x);
        if (from == From::kRest) {
            const float y = element(q[i], j);
            const Parts v = parts_of(y);
            w.a = x > y ? w.a - v.a : 0;
            w.b = x > y ? w.b - v.b : 0;
        } else if (from == From::kOthers) {
            const bool stays = mine + i * kWave * kEach + j != out;
            w.a = stays ? w.a : 0;
            w.b = stays ? w.b : 0;
        }
        return w;
    }
    // Sum of a step's elements.  They are computed here and none is kept from
    // before or for later: without this the compiler holds those of all steps,
    // more than there are registers for.
    __device__ inline Parts sum(int i, From from, std::uint32_t out)
    {
        if (from == From::kRest) {
            asm volatile("" : "+v"(p[i]), "+v"(q[i]));
        } else {
            asm volatile("" : "+v"(p[i]));
        }
        Parts s{0, 0};
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const Parts w = weight(i, j, from, out);
            s.a += w.a;
            s.b += w.b;
        }
        asm volatile("" : "+v"(s.a), "+v"(s.b));
        return s;
    }
    __device__ inline void sums(From from, std::uint32_t out, u64 (&to)[kSteps])
    {
        const auto add = [&](From f) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) to[i] = joined(sum(i, f, out));
        };
        if (from == From::kRest) {
            add(From::kRest);
        } else if (from == From::kOthers) {
            add(From::kOthers);
        } else {
            add(From::kTarget);
        }
    }

private:
    static __device__ inline float element(const u32x4& v, int j)
    {
        union {
            u32x4 v;
            T t[kEach];
        } u;
        u.v = v;
        return share(to_float(u.t[j]));
    }
};

__device__ inline u64 wave_sum(u64 x)
{
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) x += __shfl_xor(x, k);
    return x;
}
// Sums of 1 or 4 numbers over the wave: a quarter of it ends up with each.  At
// the first two steps a lane passes on the half that is not its quarter's, so
// that four cost seven exchanges and not 24.
__device__ inline u64 wave_sums(const u64 (&x)[1]) { return wave_sum(x[0]); }
__device__ inline u64 wave_sums(const u64 (&x)[4])
{
    const int lane = threadIdx.x % kWave;
    const bool upper = (lane & 32) != 0, odd = (lane & 16) != 0;
    u64 a = upper ? x[2] : x[0], b = upper ? x[3] : x[1];
    a += __shfl_xor(upper ? x[0] : x[2], 32);
    b += __shfl_xor(upper ? x[1] : x[3], 32);
    u64 s = (odd ? b : a) + __shfl_xor(odd ? a : b, 16);
#pragma unroll
    for (int k = 1; k < 16; k *= 2) s += __shfl_xor(s, k);
    return s;
}
__device__ inline u64 wave_upto(u64 x)
{
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) {
        const u64 y = __shfl_up(x, k);
        x += lane >= k ? y : 0;
    }
    return x;
}

// How far a sequence's drafts stay; a wave tests 64 of them at a time.
template <typename T>
__device__ inline int4 accept(const Verify& a, const Rows& r)
{
    const int lane = threadIdx.x % kWave, drafts = r.count - 1;
    for (int base = 0; base < drafts; base += kWave) {
        const int i = base + lane;
        bool stays = true, known = false;
        std::int32_t x = 0;
        if (i < drafts) {
            const std::int64_t row = r.begin + i;
            x = a.tokens[row + 1];
            known = static_cast<std::uint32_t>(x) < a.vocab;
            const std::int64_t at = known ? x : 0;
            const double p = share(to_float(static_cast<const T*>(a.target)[row * a.target_stride + at]));
            const double q =
                a.draft == nullptr ? 1.0 : share(to_float(static_cast<const T*>(a.draft)[row * a.draft_stride + at]));
            stays = known && static_cast<double>(a.uniform[row]) * q < p;
        }
        const u64 gone = __ballot(!stays);
        if (gone != 0) {
            const int at = __ffsll(gone) - 1;
            return int4{base + at, __shfl(known ? 1 : 0, at), __shfl(x, at), 0};
        }
    }
    return int4{drafts, 0, 0, 0};
}

// The number that is drawn, of `sum` whole numbers.
__device__ inline u64 drawn_of(float uniform, u64 sum)
{
    const float u = share(uniform) * 0x1p31f;
    const u64 k31 = u >= 0x1p31f ? 0x7fffffffull : static_cast<u64>(u);
    return k31 * (sum >> 31) + ((k31 * (sum & 0x7fffffffull)) >> 31);
}

// The element of a wave's region whose running sum passes `left`: the step,
// then the lane, then the element.
template <typename T, int kSteps>
__device__ inline std::int32_t walk(Region<T, kSteps>& x, std::uint32_t region, u64 left, From from, std::uint32_t out)
{
    constexpr int kEach = Region<T, kSteps>::kEach;
    u64 to[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) to[i] = joined(x.sum(i, from, out));
#pragma unroll
    for (int i = 0; i < kSteps; ++i) to[i] = wave_upto(to[i]);
    Region<T, 1> one;
    int step = -1;
    u64 upto = 0;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const u64 all = __shfl(to[i], kWave - 1);
        if (step < 0 && left < all) {
            step = i;
            upto = to[i];
            one.p[0] = x.p[i];
            if (from == From::kRest) one.q[0] = x.q[i];
        }
        left -= step < 0 ? all : 0;
    }
    if (step < 0) {
        return -1;
    }
    one.mine = x.mine + step * kWave * kEach;
    u64 weight[kEach], sofar = upto;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        weight[j] = joined(one.weight(0, j, from, out));
        sofar -= weight[j];
    }
    int at = 0;  // elements whose running sum does not pass it
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        sofar += weight[j];
        at += sofar <= left ? 1 : 0;
    }
    const int lane = __ffsll(__ballot(upto > left)) - 1;
    return static_cast<std::int32_t>(((region * kSteps + step) * kWave + lane) * kEach) + __shfl(at, lane);
}

// One wave draws from P alone, a row at a time: where nothing is left of it
// without the draft's, which only rows that are no distributions bring about.
template <typename T>
__device__ std::int32_t draw_full(const Verify& a, std::int64_t row, float uniform)
{
    constexpr std::uint32_t kStep = kWave * 16 / sizeof(T);
    const std::uint32_t regions = (a.vocab + kStep - 1) / kStep;
    u64 sum = 0, left = 0;
    for (int pass = 0; pass < 2; ++pass) {
        for (std::uint32_t i = 0; i < regions; ++i) {
            Region<T, 1> x;
            x.load(a, row, From::kTarget, i);
            const u64 c = wave_sum(joined(x.sum(0, From::kTarget, 0)));
            if (pass == 0) {
                sum += c;
            } else if (left < c) {
                return walk<T, 1>(x, i, left, From::kTarget, 0);
            } else {
                left -= c;
            }
        }
        if (sum == 0) break;
        left = drawn_of(uniform, sum);
    }
    return -1;
}

// One wave writes what a sequence gains; `mine` is the drafted token after row
// `lane` of it.
__device__ inline void give(const Verify& a, std::uint32_t s, const Rows& r, const int4& state, std::int32_t mine,
                            std::int32_t token)
{
    const int lane = threadIdx.x % kWave;
    for (int i = lane; i < r.count; i += kWave) {
        const std::int32_t x = i == lane ? mine : i < state.x ? a.tokens[r.begin + i + 1] : 0;
        a.out[r.begin + i] = i < state.x ? x : i == state.x ? token : -1;
    }
    if (lane == 0) {
        a.gained[s] = state.x + 1;
        if (a.lens != nullptr) a.out_lens[s] = a.lens[s] - (r.count - 1 - state.x);
    }
}
__device__ inline std::int32_t drafted(const Verify& a, const Rows& r)
{
    const int lane = threadIdx.x % kWave;
    return lane + 1 < r.count ? a.tokens[r.begin + lane + 1] : 0;
}
// One wave for a sequence without rows, or (s == seqs) for rows of no sequence.
__device__ inline void give_nothing(const Verify& a, std::uint32_t s)
{
    const int lane = threadIdx.x % kWave;
    if (s == a.seqs) {
        const std::int64_t from = a.first == nullptr || a.seqs == 0 ? 0 : a.first[0];
        const std::int64_t to = a.seqs == 0 ? 0 : a.first == nullptr ? a.seqs : a.first[a.seqs];
        for (std::int64_t i = lane; i < from && i < a.rows; i += kWave) a.out[i] = -1;
        for (std::int64_t i = (to > 0 ? to : 0) + lane; i < a.rows; i += kWave) a.out[i] = -1;
        return;
    }
    // rows past the batch, or left out
    const std::int64_t begin = a.first == nullptr ? s : a.first[s];
    const std::int64_t end = a.first == nullptr ? begin + 1 : a.first[s + 1];
    for (std::int64_t i = (begin > 0 ? begin : 0) + lane; i < end && i < a.rows; i += kWave) a.out[i] = -1;
    if (lane == 0) {
        a.gained[s] = 0;
        if (a.lens != nullptr) {
            const std::int32_t len = a.lens[s];
            const bool out = begin < end && len < end - begin;
            a.out_lens[s] = !out ? len - static_cast<std::int32_t>(end - begin) : a.stored != nullptr ? a.stored[s] : len;
        }
    }
}

// One wave sums kSteps consecutive KiB of a row, a region each, and finds how
// far the drafts stay by itself first: the same few loads for all of a
// sequence's waves, cheaper than a launch or a barrier.  Sums of whole numbers
// need no order, so nothing is shared between waves.  64 sequences of 4 drafts over
// 151,936 tokens in f32 (69 MB, as some keep all drafts and need no q) take 14.4
// us, 4.8 TB/s, on rows that the last-level cache holds, 17.1 on others, and 29.3
// just after 256 MB of writes, which then leave it; in bf16 11.2, 13.0 and 17.3, of half
// the waves behind the same trips; a single one over 32,000 3.5, the trips to its
// offsets, its tokens, their probabilities and the row.
template <typename T, int kSteps>
__global__ __launch_bounds__(kThreads) void k_verify_sum(Verify a)
{
    constexpr std::uint32_t kRegions = kThreads / kWave * kSteps;  // of a workgroup
    const std::uint32_t groups = (a.regions + kRegions - 1) / kRegions;
    const std::uint32_t s = blockIdx.x / groups;
    const std::uint32_t part = __builtin_amdgcn_readfirstlane(blockIdx.x % groups * (kThreads / kWave) + threadIdx.x / kWave);
    const Rows r = rows_of(a, s);
    const bool first = threadIdx.x % kWave == 0;
    if (r.count == 0 || part * kSteps >= a.regions) {
        if (part == 0 && first) a.state[s].count = 0;
        return;
    }
    const float uniform = a.uniform[r.begin + r.count - 1];
    const int4 state = accept<T>(a, r);
    Region<T, kSteps> x;
    x.load(a, r.begin + state.x, from_of(a, state), part);
    u64 sum[kSteps];
    x.sums(from_of(a, state), state.z, sum);
    const u64 mine = wave_sums(sum);
    const std::uint32_t region = part * kSteps + threadIdx.x % kWave / (kWave / kSteps);
    if (threadIdx.x % (kWave / kSteps) == 0 && region < a.regions) {
        a.sums[static_cast<std::size_t>(s) * a.regions + region] = mine;
    }
    if (part == 0 && first) {
        const std::int32_t count = length_of(a, s) < r.count ? 0 : r.count;
        a.state[s] = State{state, static_cast<std::int32_t>(r.begin), count, uniform};
    }
}

// One wave per sequence: the region whose running sum passes the drawn number,
// and the element in it.  The last wave clears the rows of no sequence.  4.3 us
// for those 64, 3.5 for the one: trips to the sums and to the region, and scans.
template <typename T>
__global__ __launch_bounds__(kWave) void k_verify_find(Verify a)
{
    constexpr int kHeld = 12;  // regions of a lane that stay in registers
    const std::uint32_t s = blockIdx.x;
    const int lane = threadIdx.x;
    State own_state{};
    if (s < a.seqs) own_state = a.state[s];
    if (own_state.count == 0) {
        give_nothing(a, s);
        return;
    }
    const Rows r{own_state.begin, own_state.count};
    const float uniform = own_state.uniform;
    const int4 state = own_state.drafts;
    const std::int32_t mine = drafted(a, r);
    const From from = from_of(a, state);
    const u64* sums = a.sums + static_cast<std::size_t>(s) * a.regions;
    const std::uint32_t each = (a.regions + kWave - 1) / kWave;
    const std::uint32_t begin = lane * each < a.regions ? lane * each : a.regions;
    const std::uint32_t end = begin + each < a.regions ? begin + each : a.regions;
    u64 held[kHeld], own = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) held[i] = begin + i < end ? sums[begin + i] : 0;
#pragma unroll
    for (int i = 4; i < kHeld; ++i) held[i] = 0;
    if (each > 4) {
#pragma unroll
        for (int i = 4; i < kHeld; ++i) held[i] = begin + i < end ? sums[begin + i] : 0;
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) own += held[i];
#pragma unroll 4
    for (std::uint32_t i = begin + kHeld; i < end; ++i) own += sums[i];
    const u64 upto = wave_upto(own), sum = __shfl(upto, kWave - 1);
    std::int32_t token = -1;
    if (sum != 0) {
        const u64 k = drawn_of(uniform, sum);
        const int owner = __ffsll(__ballot(upto > k)) - 1;
        // what is left of k in the owner's regions, and the one that it is in
        u64 left = k - (upto - own);
        std::uint32_t region = begin;
        bool found = false;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            found |= left < held[i];
            left -= found ? 0 : held[i];
            region += found ? 0 : 1;
        }
        if (lane == owner && !found) {
            for (; region < end && left >= sums[region]; ++region) left -= sums[region];
        }
        region = __builtin_amdgcn_readfirstlane(__shfl(region, owner));
        left = __shfl(left, owner);
        Region<T, 1> x;
        x.load(a, r.begin + state.x, from, region);
        token = walk<T, 1>(x, region, left, from, state.z);
    } else {
        token = draw_full<T>(a, r.begin + state.x, uniform);
    }
    give(a, s, r, state, mine, token);
}

// All of it in one workgroup per sequence, for rows that its registers hold:
// the row is read once and one barrier passed.  The last workgroup clears the
// rows of no sequence.  64 sequences over 4,000 tokens take 6.1 us.
template <typename T, int kSteps>
__global__ __launch_bounds__(1024) void k_verify_one(Verify a)
{
    __shared__ u64 s_sum[16];
    const std::uint32_t s = blockIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), waves = static_cast<int>(blockDim.x) / kWave;
    Rows r{0, 0};
    if (s < a.seqs) r = rows_of(a, s);
    if (r.count == 0) {
        if (wave == 0) give_nothing(a, s);
        return;
    }
    const std::int32_t len = length_of(a, s);  // by every wave before one may write over it
    const float uniform = a.uniform[r.begin + r.count - 1];
    const std::int32_t mine = drafted(a, r);
    const int4 state = accept<T>(a, r);
    const From from = from_of(a, state);
    Region<T, kSteps> x;
    x.load(a, r.begin + state.x, from, wave);
    u64 step[kSteps], own = 0;
    x.sums(from, state.z, step);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) own += step[i];
    own = wave_sum(own);
    if (threadIdx.x % kWave == 0) s_sum[wave] = own;
    __syncthreads();
    if (len < r.count) {
        if (wave == 0) give_nothing(a, s);
        return;
    }
    u64 sum = 0;
    for (int i = 0; i < waves; ++i) sum += s_sum[i];
    if (sum == 0) {
        if (wave == 0) give(a, s, r, state, mine, draw_full<T>(a, r.begin + state.x, uniform));
        return;
    }
    u64 left = drawn_of(uniform, sum);
    for (int i = 0; i < wave; ++i) {  // another wave's, if it lies before this one's
        if (left < s_sum[i]) return;
        left -= s_sum[i];
    }
    if (left < own) give(a, s, r, state, mine, walk<T, kSteps>(x, wave, left, from, state.z));
}

// ---- host -----------------------------------------------------------------

constexpr std::uint32_t kMostVocab = 1u << 22;

// How a call is cut: from its sizes alone (by graph replays, floats unless it
// says bf16).
// A workgroup per sequence where 16 waves of two loads each hold the row: 1 and
// 256 sequences over 4,000 tokens take 5.1 and 6.3 us against 6.8 and 8.2 in two
// launches, over 8,000 7.3 and 8.0 against 6.8 and 8.7, and one launch less costs
// the host 3 us less.  Eight loads a wave would hold 32,000, but one compute unit
// then reads for 12 us what two launches are done with in 6.
// Two launches otherwise, a load a wave where few waves would be left: 64
// sequences over 16,000 take 8.1 us with one load and 8.4 with four (1,000
// waves), over 32,000 9.4 and 8.9, over 60,000 13.0 and 10.4, over 151,936 22.1
// and 17.6-18.5.
// In bf16 a workgroup each takes 7.5 us for 64 over 4,000 against 8.4 in two
// launches, 8.0 and 8.4 over 8,000, but 9.8 and 8.6 over 16,000 (1 over 16,000:
// 8.1 and 7.4), where the host's call is still the shorter, 12 us and 14.5; a
// load a wave and four: 64 over 32,000 8.9 and 9.7, over 60,000 10.8 and 10.3, over
// 151,936 17.1 and 15.4.
struct Cut {
    bool one;   // a workgroup per sequence
    int steps;  // regions of a wave
    std::uint32_t regions;
    std::size_t sums, bytes;
};
Cut cut_of(std::uint32_t seqs, std::uint32_t vocab, std::uint32_t type)
{
    const std::uint32_t each = type == HBFSIM_AMD_KV_F32 ? 256 : 512;  // elements of a step
    Cut k{};
    k.one = vocab <= 16 * 2 * each;
    if (k.one) {
        k.steps = 2;
    } else {
        const std::uint64_t waves = static_cast<std::uint64_t>(seqs) * ((vocab + 4 * each - 1) / (4 * each));
        k.steps = waves < 1500 ? 1 : 4;
    }
    k.regions = (vocab + each - 1) / each;
    if (!k.one) {
        k.sums = up256(static_cast<std::size_t>(seqs) * sizeof(State));
        k.bytes = k.sums + static_cast<std::size_t>(seqs) * k.regions * sizeof(u64);
    }
    return k;
}

bool sizes_ok(std::uint32_t seqs, std::uint32_t vocab, std::uint32_t type)
{
    return vocab != 0 && vocab <= kMostVocab && type <= HBFSIM_AMD_KV_F32 && seqs <= 0x7fffff00u;
}

template <typename T, int kSteps>
void launch_two(const Verify& a, hipStream_t s)
{
    constexpr std::uint32_t kWaves = kThreads / kWave;
    if (a.seqs != 0) {
        const dim3 groups(a.seqs * ((a.regions + kWaves * kSteps - 1) / (kWaves * kSteps)));
        hipLaunchKernelGGL((k_verify_sum<T, kSteps>), groups, dim3(kThreads), 0, s, a);
    }
    hipLaunchKernelGGL(k_verify_find<T>, dim3(a.seqs + 1), dim3(kWave), 0, s, a);
}
template <typename T>
void launch(const Verify& a, const Cut& k, hipStream_t s)
{
    if (k.one) {
        hipLaunchKernelGGL((k_verify_one<T, 2>), dim3(a.seqs + 1), dim3((k.regions + 1) / 2 * kWave), 0, s, a);
    } else if (k.steps == 1) {
        launch_two<T, 1>(a, s);
    } else {
        launch_two<T, 4>(a, s);
    }
}

}  // namespace

#define HBF_API extern "C" __attribute__((visibility("default")))

HBF_API int hbfsim_amd_verify_workspace(uint32_t seqs, uint32_t vocab, uint32_t type, size_t* bytes)
{
    if (!sizes_ok(seqs, vocab, type) || bytes == nullptr) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    *bytes = seqs == 0 ? 0 : cut_of(seqs, vocab, type).bytes;
    return HBFSIM_OK;
}

HBF_API int hbfsim_amd_verify_step(const void* d_target, const void* d_draft, uint32_t type, uint32_t vocab,
                                   int64_t target_stride, int64_t draft_stride, const int32_t* d_tokens,
                                   const float* d_uniform, const int32_t* d_first, uint32_t seqs, uint32_t tokens,
                                   const int32_t* d_lens, const int32_t* d_stored, int32_t* d_out, int32_t* d_gained,
                                   int32_t* d_out_lens, void* d_workspace, size_t workspace_bytes, void* stream)
{
    if (!sizes_ok(seqs, vocab, type) || tokens > 0x7fffff00u || (d_first == nullptr && tokens != seqs)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (seqs == 0 && tokens == 0) {
        return HBFSIM_OK;
    }
    const Cut k = cut_of(seqs, vocab, type);
    if ((tokens != 0 && d_out == nullptr) ||
        (seqs != 0 && d_gained == nullptr) ||
        (seqs != 0 && k.bytes != 0 && (workspace_bytes < k.bytes || d_workspace == nullptr || !aligned16(d_workspace))) ||
        (d_lens == nullptr) != (d_out_lens == nullptr) || (d_lens == nullptr && d_stored != nullptr)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    const std::size_t out = static_cast<std::size_t>(tokens) * 4;
    if (seqs != 0 && tokens != 0 &&
        (d_target == nullptr || d_uniform == nullptr || (d_first != nullptr && d_tokens == nullptr))) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    const std::size_t each_seq = static_cast<std::size_t>(seqs) * 4;
    const auto meets_input = [&](const std::int32_t* p, std::size_t n) {
        return meet(p, n, d_tokens, out) || meet(p, n, d_uniform, out) || meet(p, n, d_first, each_seq + 4);
    };
    const auto meets_lengths = [&](const std::int32_t* p, std::size_t n) {
        return meet(p, n, d_lens, each_seq) || meet(p, n, d_stored, each_seq);
    };
    // the lengths that remain may be written over either of the given ones, place for place
    const auto over = [&](const std::int32_t* q) { return d_out_lens != q && meet(d_out_lens, each_seq, q, each_seq); };
    if (meets_input(d_out, out) || meets_lengths(d_out, out) || meets_input(d_gained, each_seq) ||
        meets_lengths(d_gained, each_seq) || meets_input(d_out_lens, each_seq) || over(d_lens) || over(d_stored) ||
        meet(d_out, out, d_gained, each_seq) || meet(d_out, out, d_out_lens, each_seq) ||
        meet(d_gained, each_seq, d_out_lens, each_seq)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    Verify a{};
    a.regions = k.regions;
    const std::uint64_t part = 4 * static_cast<std::uint64_t>(k.steps);
    if (seqs * ((k.regions + part - 1) / part) > (k.one ? kMostGroups : 4 * kMostGroups)) {
        return HBFSIM_UNSUPPORTED;
    }
    const std::int64_t each = type == HBFSIM_AMD_KV_F32 ? 4 : 8;
    a.target = d_target;
    a.draft = d_draft;
    a.target_stride = target_stride;
    a.draft_stride = draft_stride;
    a.vector = aligned16(d_target) && target_stride % each == 0 &&
                       (d_draft == nullptr || (aligned16(d_draft) && draft_stride % each == 0))
                   ? 1
                   : 0;
    a.tokens = d_tokens;
    a.uniform = d_uniform;
    a.first = d_first;
    a.lens = d_lens;
    a.stored = d_stored;
    a.seqs = seqs;
    a.rows = tokens;
    a.vocab = vocab;
    a.out = d_out;
    a.gained = d_gained;
    a.out_lens = d_out_lens;
    unsigned char* ws = static_cast<unsigned char*>(d_workspace);
    a.state = reinterpret_cast<State*>(ws);
    a.sums = k.one || seqs == 0 ? nullptr : reinterpret_cast<u64*>(ws + k.sums);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == HBFSIM_AMD_KV_BF16) {
        launch<Bf16>(a, k, s);
    } else if (type == HBFSIM_AMD_KV_F16) {
        launch<F16>(a, k, s);
    } else {
        launch<float>(a, k, s);
    }
    return checked(hipGetLastError());
}

HBF_API int hbfsim_amd_verify(const void* d_target, const void* d_draft, uint32_t type, uint32_t vocab,
                              int64_t target_stride, int64_t draft_stride, const int32_t* d_tokens,
                              const float* d_uniform, const int32_t* d_first, uint32_t seqs, uint32_t tokens,
                              const int32_t* d_lens, int32_t* d_out, int32_t* d_gained, int32_t* d_out_lens,
                              void* d_workspace, size_t workspace_bytes, void* stream)
{
    return hbfsim_amd_verify_step(d_target, d_draft, type, vocab, target_stride, draft_stride, d_tokens, d_uniform,
                                  d_first, seqs, tokens, d_lens, nullptr, d_out, d_gained, d_out_lens, d_workspace,
                                  workspace_bytes, stream);
}
