// Log probabilities of rows of logits: given tokens, the entropy, the likeliest tokens.
// One pass over the logits. With d = (x - m) c, c = scale log2(e) and a running maximum m
// of its own, every lane keeps S = sum 2^d and D = sum 2^d d; another maximum m' makes
// them f S and f (D + (m - m') c S), f = 2^((m - m') c), so that lanes, waves, and the
// parts of a row that is split over blocks are joined in the same way. Then
//   log p(t) = (x_t - m) scale - ln S,   H = ln S - ln 2 D / S.
// The difference is made before the product with c: near the maximum it is exact.
//
// Likeliest tokens. A value and its token are one 64-bit key (larger values first, of
// equal ones the lower token), so that all keys differ and the k largest are one set in
// one order. The k-th largest of 64 groups' running maxima is a bound that a handful of the
// logits read so far pass (64 ln (64 / (64 - k)) of random ones): it is made at chunks 0,
// 2, 4, 8 .. of a block's part of the row, and what passes it goes to a list in LDS,
// which is sorted by counting at the end. A list that runs full (thousands of equal logits,
// or rising ones) is made again from the lanes' largest keys.
//
// Rows are split over blocks where they are few, and the parts, sums and k keys each, joined
// in the launch by the last of them, or by a second one (one row without likeliest tokens:
// 5.2 and 7.8 us).
//
// Bound: HBM where rows are many (a logit is read once, 16 bytes a lane, the next chunk
// requested before one is used; with entropy a logit costs 10 VALU slots, four of them its
// exponential), a chain of round trips where they are few. MI355X, rows of 151936: 1000 of
// bf16 without likeliest tokens 52 us (5.9 TB/s), with 1 of them 61, with 20 74; 1000 of
// fp32 with 1 91 us (6.7); 64 of fp32 with 5 15.7; one with 20 8.8, of which loads and sums
// are 0.8, the bound and the list 2.2, the part's record and arrival 0.8, the join 3.5.
// 32 logits of bf16 to a lane and chunk instead of 16, or more registers otherwise, leave 4
// to 6 waves to a SIMD instead of 8: 76 us with 1, 127 with 20.
#include "jh_common.hpp"

namespace jh {
namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kLane = 16;                  // logits of a chunk that a lane takes
constexpr int kChunk = kThreads * kLane;
constexpr int kTop = JH_LOGPROBS_TOP;
constexpr int kRoom = 1024;                // keys: the largest so far and those that enter
constexpr int kParts = 64;                 // most parts of a row

__device__ __forceinline__ float ninf() { return -__builtin_inff(); }

// 0 is below all keys (NaN and -inf, which are never among the likeliest).
__device__ __forceinline__ uint64_t key_of(float v, int i) {
    const uint32_t u = __float_as_uint(v + 0.0f);  // (-0 is 0)
    const uint64_t k = (uint64_t)((u & 0x80000000u) ? ~u : u | 0x80000000u) << 32 | (uint32_t)~i;
    return v > ninf() ? k : 0;
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return key ? __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u) : ninf();
}
__device__ __forceinline__ int token_of(uint64_t key) { return (int)~(uint32_t)key; }

__device__ __forceinline__ uint64_t wave_max_key(uint64_t k) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = (uint64_t)(uint32_t)__shfl_xor((int)(k >> 32), d, 64) << 32 | (uint32_t)__shfl_xor((int)k, d, 64);
        k = k > o ? k : o;
    }
    return k;
}

template <int CTRL>
__device__ __forceinline__ int dpp_of(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, false);
}
template <int CTRL>
__device__ __forceinline__ float dpp_of(float x) {
    return __builtin_bit_cast(float, dpp_of<CTRL>(__builtin_bit_cast(int, x)));
}
// Over each 4 lanes.
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, dpp_of<0xB1>(v));         // quad_perm [1,0,3,2]
    return fmaxf(v, dpp_of<0x4E>(v));      // quad_perm [2,3,0,1]
}

// Sums of e^(scale (x - m)), as above.
struct Sums {
    float m, s, d;
};
__device__ __forceinline__ void move_to(Sums& a, float m, float c) {
    const float by = (a.m - m) * c, f = __builtin_amdgcn_exp2f(by);
    a.d = f > 0.0f ? f * fmaf(by, a.s, a.d) : 0.0f;  // (nothing is left: by may be -inf)
    a.s *= f;
    a.m = m;
}

__device__ __forceinline__ float load_logit(const LogProbsArgs& a, int64_t row, int i) {
    const int64_t at = row * a.stride + i;
    return a.f32 ? static_cast<const float*>(a.x)[at] : bf16_to_f32(static_cast<const uint16_t*>(a.x)[at]);
}

// The logit of token `id` of a row, NaN for none.
__device__ __forceinline__ float logit_of(const LogProbsArgs& a, int64_t row, int id) {
    return (uint32_t)id < (uint32_t)a.vocab ? load_logit(a, row, id) : __builtin_nanf("");
}

// What is known of a row when all of it has been read.
// given: the logit of the thread's token.
__device__ __forceinline__ float finish_row(const LogProbsArgs& a, int64_t row, const Sums& t, float given, int tid) {
    // (no distribution: a NaN among the terms, or a maximum that is not finite)
    const float ln = t.m > ninf() && t.m < __builtin_inff() ? logf(t.s) : __builtin_nanf("");
    if (tid < a.n_tokens) a.logprobs[row * a.n_tokens + tid] = (given - t.m) * a.scale - ln;
    if (tid == 0 && a.entropy) a.entropy[row] = ln - kLn2 * t.d / t.s;
    return ln;
}
// The row's likeliest tokens, from its `n` largest keys in order; the lowest tokens that are
// not among them where there are fewer than are asked for (all others are NaN or -inf).
__device__ __forceinline__ void finish_top(const LogProbsArgs& a, int64_t row, const Sums& t, float ln, const uint64_t* keys,
                                           int n, int tid) {
    if (tid >= a.top_k) return;
    int id = 0;
    float v = ninf();
    if (tid < n) {
        id = token_of(keys[tid]), v = value_of(keys[tid]);
    } else {
        int left = tid - n;  // so many free tokens come before
        for (id = 0;; id++) {
            bool taken = false;
            for (int i = 0; i < n; i++) taken |= token_of(keys[i]) == id;
            if (!taken && left-- == 0) break;
        }
    }
    a.top_ids[row * a.top_k + tid] = id;
    a.top_logprobs[row * a.top_k + tid] = (v - t.m) * a.scale - ln;
}

// How many of n keys in LDS are above `mine`, counted by 8 lanes (in each of them).
__device__ __forceinline__ int count_above(const uint64_t* keys, int n, uint64_t mine) {
    int above = 0;
#pragma unroll 2
    for (int j = threadIdx.x & 7; j < n; j += 8) above += keys[j] > mine;
    above += dpp_of<0xB1>(above);   // quad_perm [1,0,3,2]
    above += dpp_of<0x4E>(above);   // quad_perm [2,3,0,1]
    return above + dpp_of<0x141>(above);  // row_half_mirror
}

// The `k` largest of n keys in LDS, in order, to `to`; by all threads of a block, which
// meet before and have to meet after.
template <int NT>
__device__ __forceinline__ void sort_largest(const uint64_t* keys, int n, uint64_t* to, int k) {
    for (int i0 = 0; i0 < n; i0 += NT / 8) {
        const int i = i0 + (int)threadIdx.x / 8;
        const uint64_t mine = keys[min(i, n - 1)];
        const int above = count_above(keys, n, mine);
        if (i < n && above < k && (threadIdx.x & 7) == 0) to[above] = mine;
    }
}

// A part of a row in the workspace: its sums (16 bytes), then its k largest keys in order (0
// where there are fewer). Records are whole 128-byte lines, so that no two XCDs write one.
constexpr int kLine = 128;
__host__ __device__ constexpr int record_bytes(int k) { return (16 + 8 * k + kLine - 1) / kLine * kLine; }

// A row as whole 16-byte vectors, and fewer than kEach logits before and behind them.
template <bool F32>
struct Row {
    static constexpr int kEach = F32 ? 4 : 8, kVecs = kLane / kEach;  // logits of a vector; vectors of a lane and chunk
    int head, vectors;
    __amdgpu_buffer_rsrc_t body;
    __device__ __forceinline__ Row(const LogProbsArgs& a, int64_t row) {
        const char* const p = static_cast<const char*>(a.x) + row * a.stride * (F32 ? 4 : 2);
        head = min(a.vocab, (int)((0 - (uintptr_t)p) & 15) / (F32 ? 4 : 2));
        vectors = (a.vocab - head) / kEach;
        body = make_rsrc(p + head * (F32 ? 4 : 2), (uint32_t)vectors * 16);
    }
    __device__ __forceinline__ int chunks() const { return (vectors + kChunk / kEach - 1) / (kChunk / kEach); }
    // The number of the lane's vector i of a chunk.
    __device__ __forceinline__ int at(int chunk, int i) const { return chunk * (kChunk / kEach) + i * kThreads + (int)threadIdx.x; }
    __device__ __forceinline__ int token(int chunk, int i, int j) const { return head + at(chunk, i) * kEach + j; }
    // (behind the last vector: 0)
    __device__ __forceinline__ uint4 load(int chunk, int i) const { return buf_load16_nt(body, (uint32_t)at(chunk, i) * 16); }
    // Vectors behind the last one as -inf.
    __device__ __forceinline__ uint4 trim(int chunk, int i, uint4 v) const {
        constexpr uint32_t none = F32 ? 0xFF800000u : 0xFF80FF80u;
        return at(chunk, i) < vectors ? v : make_uint4(none, none, none, none);
    }
};

// Element j of a vector's words (j need not be known when compiled).
template <bool F32>
__device__ __forceinline__ float element(uint4 v, int j) {
    const int at = F32 ? j : j >> 1;
    const uint32_t lo = at & 1 ? v.y : v.x, hi = at & 1 ? v.w : v.z, u = at & 2 ? hi : lo;
    return __uint_as_float(F32 ? u : j & 1 ? u & 0xFFFF0000u : u << 16);
}

// Logit i of a lane's share of a chunk (i need not be known when compiled).
template <bool F32>
__device__ __forceinline__ float logit_at(const uint4 (&v)[Row<F32>::kVecs], int i) {
    constexpr int kEach = Row<F32>::kEach;
    uint4 u = v[0];
#pragma unroll
    for (int n = 1; n < Row<F32>::kVecs; n++) {
        const bool here = i / kEach == n;
        u.x = here ? v[n].x : u.x, u.y = here ? v[n].y : u.y, u.z = here ? v[n].z : u.z, u.w = here ? v[n].w : u.w;
    }
    return element<F32>(u, i % kEach);
}

// Sum over the lanes up to this one.
__device__ __forceinline__ int scan64(int v) {
    auto dpp = [](int x, auto ctrl, auto rows) {
        return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    };
    using All = std::integral_constant<int, 0xF>;
    v += dpp(v, std::integral_constant<int, 0x111>{}, All{});  // row_shr:1
    v += dpp(v, std::integral_constant<int, 0x112>{}, All{});  // row_shr:2
    v += dpp(v, std::integral_constant<int, 0x114>{}, All{});  // row_shr:4
    v += dpp(v, std::integral_constant<int, 0x118>{}, All{});  // row_shr:8
    v += dpp(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row_bcast:15
    v += dpp(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row_bcast:31
    return v;
}

// f(value) of a lane's share of a chunk.
template <bool F32, class Fn>
__device__ __forceinline__ void each(const uint4 (&v)[Row<F32>::kVecs], Fn f) {
#pragma unroll
    for (int i = 0; i < Row<F32>::kVecs; i++)
#pragma unroll
        for (int j = 0; j < Row<F32>::kEach; j++) f(element<F32>(v[i], j));
}

// A block's keys.
struct Keys {
    uint64_t list[kRoom];
    uint64_t sorted[kTop];
    __attribute__((aligned(16))) float group[2][64];
    __attribute__((aligned(16))) float least[2][kWaves];
    uint64_t head[kParts];
    uint64_t wave[kWaves];
    uint64_t bound;
    int extra;       // keys of logits outside the vectors
    int entered[3];  // keys that came in behind the e-th bound and before the next: entered[e % 3]
};

// Every key of chunks first .. last - 1, one after the other.
template <bool F32, class Fn>
__device__ __forceinline__ void each_key(const Row<F32>& r, int first, int last, Fn f) {
    for (int chunk = first; chunk < last; chunk++)
#pragma unroll 1
        for (int u = 0; u < Row<F32>::kVecs; u++) {
            const uint4 v = r.trim(chunk, u, r.load(chunk, u));
#pragma unroll 1
            for (int j = 0; j < Row<F32>::kEach; j++) f(key_of(element<F32>(v, j), r.token(chunk, u, j)));
        }
}

// The list of a part (chunks first .. last - 1) that had no room for what came in, made
// again behind `have` keys: of the lanes' largest keys the k-th is a bound that the k largest
// keys pass, and with many equal logits few others, since a lane's are the lowest tokens
// first. If too many do all the same, the largest keys are taken one by one. Returns the
// list's length. By all threads.
template <bool F32>
__device__ __forceinline__ int again(Keys& s, const Row<F32>& r, int have, int first, int last, int k) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __syncthreads();  // (all have read the counts)
    uint64_t best = 0;
    each_key(r, first, last, [&](uint64_t key) { best = key > best ? key : best; });
    uint64_t* const lanes = s.list + kRoom - kThreads;
    lanes[tid] = best;
    if (tid == 0) s.entered[0] = 0, s.bound = 0;
    __syncthreads();
    int over = 0;
#pragma unroll 2
    for (int i = 0; i < kThreads; i++) over += lanes[i] > best;
    if (best && over == k - 1) s.bound = best;  // (one lane; none where fewer than k have keys)
    __syncthreads();
    const uint64_t bound = s.bound;
    each_key(r, first, last, [&](uint64_t key) {
        if (key == 0 || key < bound) return;
        const int at = have + atomicAdd(&s.entered[0], 1);
        if (at < kRoom) s.list[at] = key;
    });
    __syncthreads();
    int n = have + s.entered[0];
    if (n <= kRoom) return n;
    uint64_t below = ~0ull;
    n = have;
    for (int i = 0; i < k; i++) {
        best = 0;
        each_key(r, first, last, [&](uint64_t key) { best = key < below && key > best ? key : best; });
        best = wave_max_key(best);
        if (lane == 0) s.wave[wave] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; w++) best = best > s.wave[w] ? best : s.wave[w];
        if (best == 0) break;
        if (tid == 0) s.list[n] = best;
        n++;
        below = best;
        __syncthreads();
    }
    __syncthreads();
    return n;
}

// The parts of a row joined, by all threads of a block. L2: the records were stored by this
// launch on this XCD (device-coherent loads: past the CU's L1).
template <bool L2>
__device__ __forceinline__ void join_parts(const LogProbsArgs& a, int64_t row, int parts, const char* records, float given, Keys& s) {
    constexpr int kAux = L2 ? kAuxSc1 : 0, kEach = kParts * kTop / kThreads;
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    const int tid = threadIdx.x, lane = tid & 63, k = a.top_k, size = record_bytes(k);
    const auto r = make_rsrc(records, (uint32_t)(parts * size));
    auto key_at = [&](int p, int j) {
        return __builtin_bit_cast(uint64_t, (u32x2_t)__builtin_amdgcn_raw_buffer_load_b64(r, (uint32_t)(p * size + 16 + 8 * j), 0, kAux));
    };
    // everything at once
    const u32x4_t sums = __builtin_amdgcn_raw_buffer_load_b128(r, (uint32_t)(lane * size), 0, kAux);
    uint64_t mine[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const int i = e * kThreads + tid;
        mine[e] = i < parts * k ? key_at(i / k, i % k) : 0;
    }
    // A bound: of the parts' keys in place `at` the `count`-th largest, which has k keys
    // at or above it, and at most k * k of the parts' (kRoom holds them).
    const int at = k ? (k + parts - 1) / parts - 1 : 0, count = (k + at) / (at + 1);
    static_assert(kTop * kTop <= kRoom, "room for what passes the bound");
    const uint64_t head = k && lane < parts ? key_at(lane, at) : 0;
    const float c = a.scale * kLog2e;
    Sums t{ninf(), 0.0f, 0.0f};
    if (lane < parts) t = Sums{__uint_as_float(sums.x), __uint_as_float(sums.y), __uint_as_float(sums.z)};
    const float m = wave_max(t.m);
    if (t.m > ninf()) move_to(t, m, c);
    const Sums all{m, wave_sum(t.s), wave_sum(t.d)};
    const float ln = finish_row(a, row, all, given, tid);
    if (k == 0) return;
    if (tid < parts) s.head[tid] = head;
    if (tid == 0) s.entered[0] = 0, s.bound = ~0ull;
    __syncthreads();
    // (0 where a part among them has no key in that place)
    for (int i0 = 0; i0 < parts; i0 += kThreads / 8) {
        const int i = i0 + tid / 8;
        const uint64_t o = s.head[min(i, parts - 1)];
        if (count_above(s.head, parts, o) < count && i < parts && (tid & 7) == 0)
            atomicMin(reinterpret_cast<unsigned long long*>(&s.bound), (unsigned long long)o);
    }
    __syncthreads();
    const uint64_t least = s.bound;
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        if (e * kThreads >= parts * k) break;
        if (mine[e] && mine[e] >= least) s.list[atomicAdd(&s.entered[0], 1)] = mine[e];
    }
    __syncthreads();
    const int n = s.entered[0];
    sort_largest<kThreads>(s.list, n, s.sorted, k);
    __syncthreads();
    finish_top(a, row, all, ln, s.sorted, min(n, k), tid);
}

// Where the rows' parts meet. With arrivals, all parts of a row run on one XCD, and the one
// that arrives last joins them; without, a launch that follows does.
struct Meeting {
    int parts, per;    // parts of a row, chunks of a part
    char* records;
    int* arrivals;     // of row r: [r % 8][r / 8], zero between calls; or nullptr
};

template <bool F32, bool ENT, bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogProbsArgs a, Meeting w) {
    constexpr int kVecs = Row<F32>::kVecs;
    __shared__ Keys s;
    __shared__ Sums s_sum[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.top_k;
    const int parts = w.parts;
    // (block b runs on XCD b % 8)
    const int64_t row = w.arrivals ? blockIdx.x / (8 * parts) * 8 + blockIdx.x % 8 : blockIdx.x / parts;
    const int part = w.arrivals ? blockIdx.x / 8 % parts : blockIdx.x % parts;
    if (row >= a.rows) return;
    const Row<F32> r(a, row);
    const int first = part * w.per, last = min(r.chunks(), first + w.per);
    const float c = a.scale * kLog2e;
    Sums t{ninf(), 0.0f, 0.0f};
    int have = 0, epoch = 0;  // keys in the list before the last bound, and its number
    float bound = ninf();
    // (a token's number first, its logit behind the first chunk: nothing waits for either)
    const int id = tid < a.n_tokens ? a.tokens[row * a.n_tokens + tid] : -1;
    uint4 v[kVecs], next[kVecs];
    if (first < last)
#pragma unroll
        for (int i = 0; i < kVecs; i++) v[i] = r.load(first, i);
    // the logits before and behind the vectors: one to a lane of the row's first block
    if (part == 0 && wave == 0) {
        const int behind = r.head + r.vectors * Row<F32>::kEach, at = lane < r.head ? lane : behind + lane - r.head;
        const float x = at < a.vocab ? load_logit(a, row, at) : ninf();
        t.m = fmaxf(t.m, x);
        t.s = x == ninf() ? 0.0f : x - x + 1.0f;  // (NaN of a logit that is not finite)
        if constexpr (TOP) {
            const uint64_t key = key_of(x, at), some = __ballot(key != 0);
            if (key) s.list[__popcll(some & ((1ull << lane) - 1))] = key;
            if (lane == 0) s.extra = __popcll(some);
        }
    } else if (TOP && part != 0 && tid == 0) {
        s.extra = 0;
    }
    if constexpr (TOP) {
        if (tid < 3) s.entered[tid] = 0;
        __syncthreads();
        have = s.extra;
    }
    // the sums of a chunk; the lane's largest
    auto add = [&](int chunk) {
        if (r.at(chunk + 1, 0) - tid > r.vectors)
#pragma unroll
            for (int i = 0; i < kVecs; i++) v[i] = r.trim(chunk, i, v[i]);
        float top = ninf();
        each<F32>(v, [&](float x) { top = fmaxf(top, x); });
        if (top > t.m) {
            if (t.m > ninf()) move_to(t, top, c);
            else t.m = top;
        }
        const float m = t.m > ninf() ? t.m : 0.0f;
        each<F32>(v, [&](float x) {
            const float d = (x - m) * c, e = __builtin_amdgcn_exp2f(d);
            t.s += e;
            if constexpr (ENT) t.d = fmaf(e, fmaxf(d, -256.0f), t.d);  // (a logit of -inf adds 0)
        });
        return top;
    };
    // The k-th largest of 64 groups' maxima so far: the least of which fewer than k are above.
    // A wave looks at 16 of them, four lanes at each.
    auto make_bound = [&]() {
        float* const group = s.group[epoch & 1];
        const float g = quad_max(t.m);
        if ((lane & 3) == 0) group[tid / 4] = g;
        __syncthreads();
        int over = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 o = reinterpret_cast<const float4*>(group)[i * 4 + (lane & 3)];
            over += (o.x > g) + (o.y > g) + (o.z > g) + (o.w > g);
        }
        over += dpp_of<0xB1>(over), over += dpp_of<0x4E>(over);
        const float least = -wave_max(over < k ? -g : ninf());
        if (lane == 0) s.least[epoch & 1][wave] = least;
        __syncthreads();
        const float4 w4 = *reinterpret_cast<const float4*>(s.least[epoch & 1]);
        bound = fmaxf(fminf(fminf(w4.x, w4.y), fminf(w4.z, w4.w)), -3.402823466e38f);  // (-inf never enters)
    };
    auto push = [&](int chunk, float top) {
        if (!__any(top >= bound)) return;
        uint32_t bits = 0;  // of the lane's logits
#pragma unroll
        for (int i = 0; i < kLane; i++) bits |= logit_at<F32>(v, i) >= bound ? 1u << i : 0u;
        // places: a sum over the lanes, one addition for the wave
        const int count = __popc(bits), upto = scan64(count);
        int at = 0;
        if (lane == 63) at = atomicAdd(&s.entered[epoch % 3], upto);
        at = have + __builtin_amdgcn_readlane(at, 63) + upto - count;
        for (; bits; bits &= bits - 1, at++) {
            const int i = __ffs(bits) - 1;
            if (at < kRoom)
                s.list[at] = key_of(logit_at<F32>(v, i), r.token(chunk, i / Row<F32>::kEach, i % Row<F32>::kEach));
        }
    };
    int chunk = first;
    bool lost = false;  // more came in than the list has room for
    auto take = [&](bool bound_first) {
        if (chunk + 1 < last)
#pragma unroll
            for (int i = 0; i < kVecs; i++) next[i] = r.load(chunk + 1, i);
        const float top = add(chunk);
        if constexpr (TOP) {
            if (bound_first) make_bound();
            if (!lost) push(chunk, top);
        }
#pragma unroll
        for (int i = 0; i < kVecs; i++) v[i] = next[i];
    };
    if (first < last) take(true), chunk++;
    const float given = logit_of(a, row, id);
    for (int run = 1; chunk < last; run *= 2) {
        if (TOP && run > 1) {
            // a new bound, and what has come in since the last one counted
            epoch++;
            make_bound();
            if (tid == 0) s.entered[(epoch + 1) % 3] = 0;
            have += s.entered[(epoch + 2) % 3];
            if (have > kRoom) lost = true, have = 0;
        }
        for (const int to = min(last, chunk + run); chunk < to; chunk++) take(false);
    }
    // lanes, then waves
    const float m = wave_max(t.m);
    if (t.m > ninf()) move_to(t, m, c);
    t.s = wave_sum(t.s), t.d = wave_sum(t.d);
    if (lane == 0) s_sum[wave] = Sums{m, t.s, t.d};
    __syncthreads();
    if constexpr (TOP) {
        have += s.entered[epoch % 3];
        if (lost || have > kRoom) have = again(s, r, s.extra, first, last, k);
        sort_largest<kThreads>(s.list, have, s.sorted, k);
        have = min(have, k);
        __syncthreads();
    }
    Sums all{ninf(), 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; w++) all.m = fmaxf(all.m, s_sum[w].m);
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        Sums u = s_sum[w];
        if (u.m > ninf()) move_to(u, all.m, c);
        all.s += u.s, all.d += u.d;
    }
    if (parts == 1) {
        const float ln = finish_row(a, row, all, given, tid);
        if constexpr (TOP) finish_top(a, row, all, ln, s.sorted, have, tid);
        return;
    }
    char* const records = w.records + row * parts * record_bytes(k);
    char* const to = records + part * record_bytes(k);
    if (tid == 0) *reinterpret_cast<float4*>(to) = make_float4(all.m, all.s, all.d, 0.0f);
    if (TOP && tid < k) reinterpret_cast<uint64_t*>(to + 16)[tid] = tid < have ? s.sorted[tid] : 0;
    if (!w.arrivals) return;
    // The records' stores are done before the arrival is counted in the XCD's L2, and are read
    // past this CU's L1 after it.
    __shared__ int s_last;
    wait_vmem<0>();
    __syncthreads();
    int* const arrivals = w.arrivals + row % 8 * kLogProbsRows + row / 8;
    if (tid == 0) s_last = __hip_atomic_fetch_add(arrivals, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    __syncthreads();
    if (!s_last) return;
    join_parts<true>(a, row, parts, records, given, s);
    if (tid == 0) __hip_atomic_store(arrivals, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogProbsArgs a, int parts, const char* records) {
    __shared__ Keys s;
    const int64_t row = blockIdx.x;
    const float given = (int)threadIdx.x < a.n_tokens ? logit_of(a, row, a.tokens[row * a.n_tokens + threadIdx.x]) : 0.0f;
    join_parts<false>(a, row, parts, records + row * parts * record_bytes(a.top_k), given, s);
}

// Parts of a row and the chunks of each. Up to six blocks of 256 threads to a CU (of eight
// that find room) fill HBM, and a part's end and its joining cost what reading a few chunks
// does: 1000 rows of 151936 bf16 logits 63 us as 1000 blocks, 66 as 2000; 300 of them 33 as
// 1200 blocks, 31 as 1500, 35 as 2100.
Meeting meeting_of(const LogProbsArgs& a, int num_cus) {
    const int64_t chunks = std::max<int64_t>(1, (a.vocab + kChunk - 1) / kChunk);
    const int64_t parts = std::max<int64_t>(1, std::min({6 * (int64_t)num_cus / a.rows, chunks, (int64_t)kParts}));
    Meeting w{};
    w.per = (int)((chunks + parts - 1) / parts);
    w.parts = (int)((chunks + w.per - 1) / w.per);
    return w;
}

}  // namespace

size_t logprobs_workspace_bytes(const LogProbsArgs& a, int num_cus) {
    const Meeting w = meeting_of(a, num_cus);
    return w.parts > 1 ? (size_t)record_bytes(a.top_k) * w.parts * (size_t)a.rows : 0;
}

Status launch_logprobs(const LogProbsArgs& a, void* workspace, int num_cus, int* sync, hipStream_t st) {
    Meeting w = meeting_of(a, num_cus);
    w.records = static_cast<char*>(workspace);
    if (w.parts > 1 && a.rows <= 8 * kLogProbsRows) w.arrivals = sync;
    // (a grid holds fewer than 2^32 threads; rows that are split are few)
    constexpr int kMostRows = 1 << 23;
    static_assert((int64_t)kMostRows * kThreads < ((int64_t)1 << 32), "rows of a launch");
    auto go = [&](auto f32, auto ent, auto top) {
        for (int first = 0; first < a.rows; first += kMostRows) {
            LogProbsArgs part = a;
            part.rows = std::min(kMostRows, a.rows - first);
            part.x = static_cast<const char*>(a.x) + first * a.stride * (a.f32 ? 4 : 2);
            if (a.n_tokens) part.tokens += (int64_t)first * a.n_tokens, part.logprobs += (int64_t)first * a.n_tokens;
            if (a.entropy) part.entropy += first;
            if (a.top_k) part.top_ids += (int64_t)first * a.top_k, part.top_logprobs += (int64_t)first * a.top_k;
            const int64_t rows = w.arrivals ? ((int64_t)part.rows + 7) / 8 * 8 : part.rows;
            hipLaunchKernelGGL((logprobs_kernel<decltype(f32)::value, decltype(ent)::value, decltype(top)::value>),
                               dim3((unsigned)(rows * w.parts)), dim3(kThreads), 0, st, part, w);
        }
    };
    auto with = [&](auto f32, auto ent) { a.top_k ? go(f32, ent, std::true_type{}) : go(f32, ent, std::false_type{}); };
    auto typed = [&](auto f32) { a.entropy ? with(f32, std::true_type{}) : with(f32, std::false_type{}); };
    a.f32 ? typed(std::true_type{}) : typed(std::false_type{});
    if (w.parts > 1 && !w.arrivals)
        hipLaunchKernelGGL(logprobs_join_kernel, dim3((unsigned)a.rows), dim3(kThreads), 0, st, a, w.parts, w.records);
    return Status::ok();
}

}  // namespace jh
