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
// 24 bits, so a p above 2^-17 keeps all of them; the rounding below that, at
// most 2^-41 of the whole, is the price of sums that do not depend on their
// order) and are summed in 64 bits: vocabularies up to 2^22 fit.
#include "kvcache.hpp"

namespace {

using namespace hbfamd::kv;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr double kUnit = 0x1p40;
constexpr double kWhole = 0x1.8p52;  // whole numbers above it are its bits plus themselves

typedef unsigned long long u64;

struct Verify {
    const void* target;
    const void* draft;  // or null
    std::int64_t target_stride, draft_stride;
    const std::int32_t* tokens;
    const float* uniform;
    const std::int32_t* first;
    const std::int32_t* lens;
    std::uint32_t seqs, rows, vocab, chunks;
    std::uint32_t vector;  // rows of both may be loaded 16 bytes at a time
    std::int32_t* out;
    std::int32_t* gained;
    std::int32_t* out_lens;
    int4* state;  // [seqs]: accepted, whether a draft was refused, that draft
    u64* sums;    // [seqs][chunks][2]: of what is drawn from, and of P alone
};

// A sequence's rows, none if they do not describe the batch.
struct Rows {
    std::int64_t begin;
    std::int32_t count;
};
__device__ inline Rows rows_of(const Verify& a, std::uint32_t s)
{
    if (a.first == nullptr) {
        return Rows{static_cast<std::int64_t>(s), 1};
    }
    const std::int64_t begin = a.first[s], count = a.first[s + 1] - begin;
    if (begin < 0 || count <= 0 || begin + count > a.rows) {
        return Rows{begin, 0};
    }
    return Rows{begin, static_cast<std::int32_t>(count)};
}

__device__ inline float share(float x) { return fminf(fmaxf(x, 0.0f), 1.0f); }
__device__ inline u64 whole(float x)
{
    return static_cast<u64>(__double_as_longlong(__fma_rn(static_cast<double>(share(x)), kUnit, kWhole))) -
           static_cast<u64>(__double_as_longlong(kWhole));
}

// Elements e .. e + kEach - 1 of a row as whole numbers, 0 past its end.
template <typename T, int kEach>
__device__ inline void load_whole(const T* row, std::uint32_t e, std::uint32_t vocab, bool vector, u64 (&x)[kEach])
{
    if (vector && e + kEach <= vocab) {
        union {
            u32x4 v;
            T t[kEach];
        } u;
        u.v = *reinterpret_cast<const u32x4*>(row + e);
#pragma unroll
        for (int i = 0; i < kEach; ++i) x[i] = whole(to_float(u.t[i]));
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float f = to_float(row[e + i < vocab ? e + i : 0]);
            x[i] = e + i < vocab ? whole(f) : 0;
        }
    }
}

// What the next token is drawn from: P where no draft was refused, otherwise
// max(P - Q, 0), or P but for the refused token.
template <typename T, int kEach>
__device__ inline void load_drawn(const Verify& a, std::int64_t row, const int4& state, std::uint32_t e, u64 (&full)[kEach],
                                  u64 (&less)[kEach])
{
    load_whole<T, kEach>(static_cast<const T*>(a.target) + row * a.target_stride, e, a.vocab, a.vector != 0, full);
    if (state.y != 0 && a.draft != nullptr) {
        u64 q[kEach];
        load_whole<T, kEach>(static_cast<const T*>(a.draft) + row * a.draft_stride, e, a.vocab, a.vector != 0, q);
#pragma unroll
        for (int i = 0; i < kEach; ++i) less[i] = full[i] > q[i] ? full[i] - q[i] : 0;
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) less[i] = state.y != 0 && e + i == static_cast<std::uint32_t>(state.z) ? 0 : full[i];
    }
}

__device__ inline u64 wave_sum(u64 x)
{
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) x += __shfl_xor(x, k);
    return x;
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
            const double q = a.draft == nullptr ? 1.0 : share(to_float(static_cast<const T*>(a.draft)[row * a.draft_stride + at]));
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

// One workgroup per (sequence, chunk of kSteps * 256 16-byte loads).
template <typename T, int kSteps>
__global__ __launch_bounds__(kThreads) void k_verify_sum(Verify a)
{
    constexpr int kEach = 16 / sizeof(T);
    __shared__ int4 s_state;
    __shared__ u64 s_sum[2][kWaves];
    const std::uint32_t s = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const Rows r = rows_of(a, s);
    if (r.count == 0) {
        return;
    }
    if (wave == 0) {
        const int4 got = accept<T>(a, r);
        if (lane == 0) s_state = got;
    }
    __syncthreads();
    const int4 state = s_state;
    if (chunk == 0 && threadIdx.x == 0) a.state[s] = state;
    u64 drawn = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const std::uint32_t e = ((chunk * kSteps + i) * kThreads + threadIdx.x) * kEach;
        u64 full[kEach], less[kEach];
        if (e < a.vocab) {
            load_drawn<T, kEach>(a, r.begin + state.x, state, e, full, less);
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                drawn += less[j];
                all += full[j];
            }
        }
    }
    drawn = wave_sum(drawn);
    all = wave_sum(all);
    if (lane == 0) {
        s_sum[0][wave] = drawn;
        s_sum[1][wave] = all;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        u64 sum = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) sum += s_sum[threadIdx.x][i];
        a.sums[(static_cast<std::size_t>(s) * a.chunks + chunk) * 2 + threadIdx.x] = sum;
    }
}

// One workgroup per sequence: the chunk, then the step, the wave, the lane and
// the element whose running sum passes the drawn number.  The last workgroup
// clears the rows of no sequence.
template <typename T, int kSteps>
__global__ __launch_bounds__(kThreads) void k_verify_find(Verify a)
{
    constexpr int kEach = 16 / sizeof(T);
    __shared__ u64 s_sum[2][kWaves];
    __shared__ u64 s_step[kSteps][kWaves];
    __shared__ u64 s_left;
    __shared__ std::uint32_t s_chunk;
    __shared__ std::int32_t s_token;
    const std::uint32_t s = blockIdx.x;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    if (s == a.seqs) {
        const std::int64_t from = a.first == nullptr || a.seqs == 0 ? 0 : a.first[0];
        const std::int64_t to = a.seqs == 0 ? 0 : a.first == nullptr ? a.seqs : a.first[a.seqs];
        for (std::int64_t i = threadIdx.x; i < a.rows; i += kThreads) {
            if (i < from || i >= to) a.out[i] = -1;
        }
        return;
    }
    const Rows r = rows_of(a, s);
    if (r.count == 0) {
        if (a.first != nullptr) {  // rows that end past the batch
            for (std::int64_t i = a.first[s] + static_cast<std::int64_t>(threadIdx.x); i < a.first[s + 1] && i < a.rows; i += kThreads) {
                if (i >= 0) a.out[i] = -1;
            }
        }
        if (threadIdx.x == 0) {
            a.gained[s] = 0;
            if (a.lens != nullptr) a.out_lens[s] = a.lens[s] - (a.first[s + 1] - a.first[s]);
        }
        return;
    }
    const int4 state = a.state[s];
    const u64* sums = a.sums + static_cast<std::size_t>(s) * a.chunks * 2;
    const std::uint32_t each = (a.chunks + kThreads - 1) / kThreads;
    const std::uint32_t begin = threadIdx.x * each < a.chunks ? threadIdx.x * each : a.chunks;
    const std::uint32_t end = begin + each < a.chunks ? begin + each : a.chunks;
    u64 mine[2] = {0, 0};
    for (std::uint32_t i = begin; i < end; ++i) {
        mine[0] += sums[2 * i];
        mine[1] += sums[2 * i + 1];
    }
    u64 upto[2] = {wave_upto(mine[0]), wave_upto(mine[1])};
    if (lane == kWave - 1) {
        s_sum[0][wave] = upto[0];
        s_sum[1][wave] = upto[1];
    }
    __syncthreads();
    u64 total[2] = {0, 0};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            upto[w] += i < wave ? s_sum[w][i] : 0;
            total[w] += s_sum[w][i];
        }
    }
    const int which = total[0] != 0 ? 0 : 1;  // nothing left: from P
    const u64 sum = total[which];
    std::int32_t token = -1;
    if (sum != 0) {
        const float u = share(a.uniform[r.begin + r.count - 1]) * 0x1p31f;
        const u64 k31 = u >= 0x1p31f ? 0x7fffffffull : static_cast<u64>(u);
        const u64 k = k31 * (sum >> 31) + ((k31 * (sum & 0x7fffffffull)) >> 31);
        u64 before = upto[which] - mine[which];
        if (k >= before && k < upto[which]) {
            for (std::uint32_t i = begin; i < end; ++i) {
                const u64 c = sums[2 * i + which];
                if (k < before + c) {
                    s_chunk = i;
                    s_left = k - before;
                    break;
                }
                before += c;
            }
        }
        __syncthreads();
        const std::uint32_t chunk = s_chunk;
        const u64 left = s_left;
        u64 lane_sum[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const std::uint32_t e = ((chunk * kSteps + i) * kThreads + threadIdx.x) * kEach;
            lane_sum[i] = 0;
            if (e < a.vocab) {
                u64 full[kEach], less[kEach];
                load_drawn<T, kEach>(a, r.begin + state.x, state, e, full, less);
#pragma unroll
                for (int j = 0; j < kEach; ++j) lane_sum[i] += which == 0 ? less[j] : full[j];
            }
            const u64 got = wave_sum(lane_sum[i]);
            if (lane == 0) s_step[i][wave] = got;
        }
        __syncthreads();
        u64 at = 0;
        for (int i = 0; i < kSteps; ++i) {
            for (int w = 0; w < kWaves; ++w) {
                const u64 c = s_step[i][w];
                if (left >= at && left < at + c && w == wave) {
                    u64 own = 0;
#pragma unroll
                    for (int n = 0; n < kSteps; ++n) own = n == i ? lane_sum[n] : own;
                    const u64 sofar = at + wave_upto(own);
                    if (left < sofar && left >= sofar - own) {
                        const std::uint32_t e = ((chunk * kSteps + i) * kThreads + threadIdx.x) * kEach;
                        u64 full[kEach], less[kEach], walk = sofar - own;
                        load_drawn<T, kEach>(a, r.begin + state.x, state, e, full, less);
                        int found = -1;
#pragma unroll
                        for (int j = 0; j < kEach; ++j) {
                            walk += which == 0 ? less[j] : full[j];
                            if (found < 0 && left < walk) found = static_cast<int>(e) + j;
                        }
                        s_token = found;
                    }
                }
                at += c;
            }
        }
        __syncthreads();
        token = s_token;
    }
    for (int i = threadIdx.x; i < r.count; i += kThreads) {
        a.out[r.begin + i] = i < state.x ? a.tokens[r.begin + i + 1] : i == state.x ? token : -1;
    }
    if (threadIdx.x == 0) {
        a.gained[s] = state.x + 1;
        if (a.lens != nullptr) a.out_lens[s] = a.lens[s] - (r.count - 1 - state.x);
    }
}

// ---- host -----------------------------------------------------------------

constexpr std::uint32_t kMostVocab = 1u << 22;
constexpr int kSteps = 8;  // of f32, half as many of the two-byte types

std::uint32_t chunks_of(std::uint32_t vocab) { return (vocab + kThreads * 4 * kSteps - 1) / (kThreads * 4 * kSteps); }

std::size_t bytes_of(std::uint32_t seqs, std::uint32_t vocab)
{
    return up256(static_cast<std::size_t>(seqs) * sizeof(int4)) + static_cast<std::size_t>(seqs) * chunks_of(vocab) * 2 * sizeof(u64);
}

bool sizes_ok(std::uint32_t seqs, std::uint32_t vocab, std::uint32_t type)
{
    return vocab != 0 && vocab <= kMostVocab && type <= HBFSIM_AMD_KV_F32 && seqs <= 0x7fffff00u;
}

template <typename T>
void launch(const Verify& a, hipStream_t s)
{
    constexpr int kOf = sizeof(T) == 4 ? kSteps : kSteps / 2;
    if (a.seqs != 0) {
        hipLaunchKernelGGL((k_verify_sum<T, kOf>), dim3(a.seqs * a.chunks), dim3(kThreads), 0, s, a);
    }
    hipLaunchKernelGGL((k_verify_find<T, kOf>), dim3(a.seqs + 1), dim3(kThreads), 0, s, a);
}

// Whether [p, p + n) and [q, q + m) have a byte in common.
bool meet(const void* p, std::size_t n, const void* q, std::size_t m)
{
    const std::uintptr_t a = reinterpret_cast<std::uintptr_t>(p), b = reinterpret_cast<std::uintptr_t>(q);
    return p != nullptr && q != nullptr && n != 0 && m != 0 && a < b + m && b < a + n;
}

}  // namespace

#define HBF_API extern "C" __attribute__((visibility("default")))

HBF_API int hbfsim_amd_verify_workspace(uint32_t seqs, uint32_t vocab, uint32_t type, size_t* bytes)
{
    if (!sizes_ok(seqs, vocab, type) || bytes == nullptr) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    *bytes = seqs == 0 ? 0 : bytes_of(seqs, vocab);
    return HBFSIM_OK;
}

HBF_API int hbfsim_amd_verify(const void* d_target, const void* d_draft, uint32_t type, uint32_t vocab,
                              int64_t target_stride, int64_t draft_stride, const int32_t* d_tokens,
                              const float* d_uniform, const int32_t* d_first, uint32_t seqs, uint32_t tokens,
                              const int32_t* d_lens, int32_t* d_out, int32_t* d_gained, int32_t* d_out_lens,
                              void* d_workspace, size_t workspace_bytes, void* stream)
{
    if (!sizes_ok(seqs, vocab, type) || tokens > 0x7fffff00u || (d_first == nullptr && tokens != seqs)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (seqs == 0 && tokens == 0) {
        return HBFSIM_OK;
    }
    const std::size_t need = seqs == 0 ? 0 : bytes_of(seqs, vocab);
    if ((tokens != 0 && d_out == nullptr) ||
        (seqs != 0 && (d_gained == nullptr || workspace_bytes < need || d_workspace == nullptr || !aligned16(d_workspace))) ||
        (d_lens == nullptr) != (d_out_lens == nullptr)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    const std::size_t out = static_cast<std::size_t>(tokens) * 4;
    if (seqs != 0 && tokens != 0 &&
        (d_target == nullptr || d_uniform == nullptr || (d_first != nullptr && d_tokens == nullptr))) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    if (meet(d_out, out, d_tokens, out) || meet(d_out, out, d_uniform, out) ||
        meet(d_out, out, d_first, d_first != nullptr ? (static_cast<std::size_t>(seqs) + 1) * 4 : 0) ||
        meet(d_out, out, d_lens, static_cast<std::size_t>(seqs) * 4)) {
        return HBFSIM_INVALID_ARGUMENT;
    }
    Verify a{};
    a.chunks = chunks_of(vocab);
    if (static_cast<std::uint64_t>(seqs) * a.chunks > 4 * kMostGroups || seqs >= 4 * kMostGroups) {
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
    a.seqs = seqs;
    a.rows = tokens;
    a.vocab = vocab;
    a.out = d_out;
    a.gained = d_gained;
    a.out_lens = d_out_lens;
    unsigned char* ws = static_cast<unsigned char*>(d_workspace);
    a.state = reinterpret_cast<int4*>(ws);
    a.sums = seqs == 0 ? nullptr : reinterpret_cast<u64*>(ws + up256(static_cast<std::size_t>(seqs) * sizeof(int4)));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == HBFSIM_AMD_KV_BF16) {
        launch<Bf16>(a, s);
    } else if (type == HBFSIM_AMD_KV_F16) {
        launch<F16>(a, s);
    } else {
        launch<float>(a, s);
    }
    return checked(hipGetLastError());
}
