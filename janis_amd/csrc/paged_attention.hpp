// Parts of attention over a paged cache that its kernels share (paged_attention.hip,
// paged_tree_attention.hip): loads into LDS, the two products, the online softmax, a row
// computed again.
#pragma once

#include "jh_common.hpp"

namespace jh {
namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kUnit = 64;       // keys: splits are whole units
constexpr int kFewRows = 32;    // rows of a tile where rows are few
constexpr int kManyRows = 128;  // ... and many
// p is held as p * 2^kPShift, and a row's maximum is moved when it grew by more than
// kLazy (log2): f16 has nothing below 2^-24 and nothing past 2^16, so p is kept high
// there (a weight of 2^-27 of the largest still has all its bits).
template <bool F16>
constexpr float kPShift = F16 ? 13.0f : 0.0f;
template <bool F16>
constexpr float kLazy = F16 ? 2.0f : 8.0f;

__device__ __forceinline__ float ninf() { return -__builtin_inff(); }

template <bool F16>
__device__ __forceinline__ floatx16 mfma(uint4 a, uint4 b, floatx16 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                      0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
}

// Terms of a probability in the product with the values: together they hold it to 2^-16
// (bf16) or 2^-22 (f16), so that results of 16 bits are rounded once, at the end. One term
// is faster where rows are many (2000 tokens of 8000 bf16 keys 240 us against 328) and
// leaves bf16 results with 1.36 times the error of that one rounding (0.00226 of their size
// against 0.00166).
constexpr int kTerms = 2;

// (a, b) as N packed 16-bit terms, each the nearest to what the earlier ones left.
template <bool F16, int N>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&t)[N]) {
#pragma unroll
    for (int n = 0; n < N; n++) {
        const f32x2_t f = {a, b};
        if constexpr (F16) {
            const f16x2_t v = __builtin_convertvector(f, f16x2_t);
            t[n] = __builtin_bit_cast(uint32_t, v);
            if (n + 1 < N) a -= (float)v.x, b -= (float)v.y;
        } else {
            t[n] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2_t));
            if (n + 1 < N) a -= __uint_as_float(t[n] << 16), b -= __uint_as_float(t[n] & 0xFFFF0000u);
        }
    }
}

template <bool F16>
__device__ __forceinline__ float2 widen2(uint32_t u) {
    if constexpr (F16) {
        const f16x2_t x = __builtin_bit_cast(f16x2_t, u);
        return make_float2((float)x.x, (float)x.y);
    }
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

// 16 bytes per lane from base + off into LDS at m0 + 16 * lane. The s_nop is the five wait
// states between a VALU write of a scalar (a readlane into `base`) and its use by a load,
// which the compiler does not see in here; it covers the M0 write too.
// ONCE: data that no other block reads (non-temporal).
template <bool ONCE>
__device__ __forceinline__ void lds_fill16(const void* base, uint32_t off, uint32_t m0) {
    if constexpr (ONCE)
        asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(uniform((int64_t)base)),
                     "{m0}"(uniform((int)m0))
                     : "memory");
    else
        asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(uniform((int64_t)base)),
                     "{m0}"(uniform((int)m0))
                     : "memory");
}
// The wave's LDS reads are done (before loads into LDS overwrite what they read).
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ uint4 lds_read16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
// Four keys of one feature: in each 16 lanes, lane i's address is 4 features (8 bytes) of
// key i / 4, and lane i receives feature i of the keys 0 .. 3.
__device__ __forceinline__ uint2 lds_read_tr(const uint8_t* p) {
    return __builtin_bit_cast(
        uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)p));
}

struct Request {
    int start, n, kv;
};
__device__ __forceinline__ Request request(const PagedAttnArgs& a, int r) {
    const int cap = a.max_blocks << a.page_shift;  // at most 2^30
    const int from = a.row_starts[r], to = a.row_starts[r + 1], kv = a.kv_lens[r];
    Request q;
    q.start = min(max(from, 0), a.n_rows);
    q.n = min(max(to, q.start), a.n_rows) - q.start;
    q.kv = min(max(kv, 0), cap);
    return q;
}

// Sum over the lanes up to this one.
template <class T>
__device__ __forceinline__ T scan64(T v) {
    auto dpp = [](T x, auto ctrl, auto rows) {
        if constexpr (sizeof(T) == 8) {
            const int2 u = __builtin_bit_cast(int2, x);
            return __builtin_bit_cast(
                T, make_int2(__builtin_amdgcn_update_dpp(0, u.x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false),
                             __builtin_amdgcn_update_dpp(0, u.y, decltype(ctrl)::value, decltype(rows)::value, 0xF, false)));
        } else {
            return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
        }
    };
    v += dpp(v, std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});  // row_shr:1
    v += dpp(v, std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});  // row_shr:2
    v += dpp(v, std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});  // row_shr:4
    v += dpp(v, std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});  // row_shr:8
    v += dpp(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row_bcast:15
    v += dpp(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row_bcast:31
    return v;
}

// Keys that row `row` of the request sees.
__device__ __forceinline__ int seen(const Request& q, int row, int G) { return max(0, q.kv - q.n + row / G + 1); }

// With TREE the new tokens of a request see each other by the bits of a mask (those of a
// run longer than the mask's bits up to their own, as above): key kv - n + b by bit b.
__device__ __forceinline__ bool is_tree(const PagedAttnArgs& a, const Request& q) { return q.n <= 32 * a.mask_words; }
// Of the 32 keys from k0 on those that the row sees, as bits; `lim`: its reach.
__device__ __forceinline__ uint32_t sees32(const PagedAttnArgs& a, const Request& q, int row, int G, int k0, int lim) {
    uint32_t bits = 0xFFFFFFFFu;
    if (is_tree(a, q)) {
        const int j = k0 - (q.kv - q.n), w = j >> 5;
        const uint32_t* const m = a.mask + (int64_t)(q.start + row / G) * a.mask_words;
        // (words before the first: committed keys, which all rows see)
        const uint32_t lo = w < 0 ? 0xFFFFFFFFu : w < a.mask_words ? m[w] : 0u;
        const uint32_t hi = w + 1 < 0 ? 0xFFFFFFFFu : w + 1 < a.mask_words ? m[w + 1] : 0u;
        bits = __builtin_amdgcn_alignbit(hi, lo, (uint32_t)j & 31u);
    }
    const int left = lim - k0;
    return left >= 32 ? bits : left <= 0 ? 0u : bits & ((1u << left) - 1);
}

// ---- a row again, key by key -------------------------------------------------------
// The products meet masked keys with p = 0, where an infinity or NaN in V gives NaN, and
// p's lesser terms (of either sign) meet an infinity that the row does see. So a row
// whose result is not finite is computed again here, by one wave, in fp32 and reading
// nothing that it does not see. m is log2; the lane's features are lane + 64 e.
template <int DH, bool F16, bool TREE>
__device__ __forceinline__ void row_again(const PagedAttnArgs& a, const Request& rq, int r, int hk, int head, int token, int kb, int lim,
                                       float& m, float& l, float (&o)[DH / 64], int lane = threadIdx.x & 63) {
    const uint4* const q = reinterpret_cast<const uint4*>(a.q + token * a.q_stride + (int64_t)head * DH);
    m = ninf(), l = 0.0f;
#pragma unroll
    for (int e = 0; e < DH / 64; e++) o[e] = 0.0f;
    for (int k0 = kb; k0 < lim; k0 += 64) {
        const int key = min(k0 + lane, lim - 1);
        int page = a.tables[(int64_t)r * a.max_blocks + (key >> a.page_shift)];
        if ((uint32_t)page >= (uint32_t)a.n_pages) page = 0;
        const int64_t at = page * a.page_stride +
                           (((int64_t)hk << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * DH;
        const uint4* const k = reinterpret_cast<const uint4*>(a.k + at);
        float s = 0.0f;
#pragma unroll 4
        for (int i = 0; i < DH / 8; i++) {
            const uint4 x = q[i], y = k[i];
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 u = widen2<F16>(xs[j]), v = widen2<F16>(ys[j]);
                s = fmaf(u.x, v.x, s);
                s = fmaf(u.y, v.y, s);
            }
        }
        bool sees = k0 + lane < lim;
        if constexpr (TREE) sees = sees32(a, rq, token - rq.start, 1, k0 + (lane & 32), lim) >> (lane & 31) & 1u;
        s = sees ? s * (a.scale * kLog2e) : ninf();
        const uint64_t votes = __ballot(sees);
        const float mn = fmaxf(m, wave_max(s));
        const float sub = mn == ninf() ? 0.0f : mn, f = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - sub);
        const float p = __builtin_amdgcn_exp2f(s - sub + kPShift<F16>);  // as the products hold it
        l = l * f + wave_sum(p);
#pragma unroll
        for (int e = 0; e < DH / 64; e++) o[e] *= f;
        m = mn;
        for (int j = 0; j < min(64, lim - k0); j++) {
            if (TREE && !(votes >> j & 1u)) continue;
            const float pj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), j));
            const int64_t row = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), j) << 32) |
                                          (uint32_t)__builtin_amdgcn_readlane((int)at, j));
#pragma unroll
            for (int e = 0; e < DH / 64; e++) {
                const uint16_t v = a.v[row + lane + 64 * e];
                o[e] = fmaf(pj, F16 ? f16_to_f32(v) : bf16_to_f32(v), o[e]);
            }
        }
    }
}

__device__ __forceinline__ void store_out(const PagedAttnArgs& a, int64_t at, float v) {
    if (a.out_dt == JH_F16) static_cast<uint16_t*>(a.out)[at] = f32_to_f16(v);
    else store_y(a.out, at, v, a.out_dt);
}
__device__ __forceinline__ void store_out4(const PagedAttnArgs& a, int64_t at, float x, float y, float z, float w) {
    if (a.out_dt == JH_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(x, y, z, w);
        return;
    }
    uint32_t lo[1], hi[1];
    if (a.out_dt == JH_F16) split_pair<true, 1>(x, y, lo), split_pair<true, 1>(z, w, hi);
    else split_pair<false, 1>(x, y, lo), split_pair<false, 1>(z, w, hi);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = make_uint2(lo[0], hi[0]);
}

// Where row `row` of a request goes: element offset of its head's first feature.
template <int DH>
__device__ __forceinline__ int64_t out_at(const PagedAttnArgs& a, const Request& q, int row, int hk, int G) {
    return ((int64_t)(q.start + row / G) * a.Hq + hk * G + row % G) * DH;
}

// Tiles of keys in LDS: row `key` (of the tile) holds its DH / 8 chunks of 16 bytes,
// chunk c at place c ^ perm(key). K rows are read by 16 lanes of consecutive keys at one
// chunk, V rows by 4 keys at 64 bytes each: over 256 bytes (all banks) none meets another.
template <int DH>
__device__ __forceinline__ int perm_k(int key) { return DH == 64 ? (key >> 1) & 7 : key & 15; }
template <int DH>
__device__ __forceinline__ int perm_v(int key) { return DH == 64 ? 4 * ((key >> 1) & 1) : 4 * (key & 3); }

// A group of eight keys (they lie in one page) of one head, keys or values, into rows
// 8 g .. of the tile at `lds`: DH / 64 loads of 1 KB. `at`: bytes from the pool to the
// group's first key, or to the last that may be loaded where that is an earlier one;
// `more`: rows that follow it.
template <int DH>
struct Filler {
    static constexpr int kN = DH / 64;
    uint32_t k[kN], v[kN];  // the lane's part of the addresses in a whole group (k: of even g)
    int lane;
    __device__ __forceinline__ Filler(int lane_ = threadIdx.x & 63) : lane(lane_) {
#pragma unroll
        for (int u = 0; u < kN; u++) {
            const int row = (u * 64 + lane) / (DH / 8), place = (u * 64 + lane) % (DH / 8);
            k[u] = row * (2 * DH) + 16 * (place ^ perm_k<DH>(row));
            v[u] = row * (2 * DH) + 16 * (place ^ perm_v<DH>(row));
        }
    }
    template <bool V, bool WHOLE, bool ONCE>
    __device__ __forceinline__ void fill(const uint16_t* pool, int64_t at, int g, uint32_t lds, int more = 0) const {
        const char* const base = reinterpret_cast<const char*>(pool) + at;
#pragma unroll
        for (int u = 0; u < kN; u++) {
            // (eight keys on, perm_k changes by one bit)
            uint32_t off = V ? v[u] : k[u] ^ ((g & 1) * (16 * perm_k<DH>(8)));
            if constexpr (!WHOLE) {
                const int row = (u * 64 + lane) / (DH / 8);
                off -= max(0, row - more) * (2 * DH);
            }
            lds_fill16<ONCE>(base, off, lds + g * (16 * DH) + u * 1024);
        }
    }
};

// Bytes from a pool to key `key` of head hk; pages outside the pool give page 0.
template <int DH>
__device__ __forceinline__ int64_t key_at(const PagedAttnArgs& a, int r, int hk, int key, bool& outside) {
    int id = a.tables[(int64_t)r * a.max_blocks + (key >> a.page_shift)];
    outside = (uint32_t)id >= (uint32_t)a.n_pages;
    if (outside) id = 0;
    return 2 * (id * a.page_stride + (((int64_t)hk << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * DH);
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
}

// The lane's row of q as B fragments: step kk holds features 16 kk + 8 h .. + 8.
template <int DH>
__device__ __forceinline__ void load_q(const PagedAttnArgs& a, const Request& q, int row, int hk, int G,
                                       uint4 (&qf)[DH / 16], int lane = threadIdx.x & 63) {
    const int h = lane >> 5;
    const uint16_t* const p = a.q + (q.start + row / G) * a.q_stride + (int64_t)(hk * G + row % G) * DH + 8 * h;
#pragma unroll
    for (int kk = 0; kk < DH / 16; kk++) qf[kk] = *reinterpret_cast<const uint4*>(p + 16 * kk);
}

// S^T of 32 keys (their rows in LDS at kt) and the wave's 32 rows.
template <int DH, bool F16>
__device__ __forceinline__ floatx16 scores32(const uint8_t* kt, const uint4 (&qf)[DH / 16], int lane = threadIdx.x & 63) {
    const int h = lane >> 5, c = lane & 31;
    const uint8_t* const row = kt + c * (2 * DH);
    const int x = (h ^ perm_k<DH>(c)) * 16;
    floatx16 s;
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < DH / 16; kk++) s = mfma<F16>(lds_read16(row + (x ^ (32 * kk))), qf[kk], s);
    return s;
}

// O^T += V^T P^T over 16 keys (their rows in LDS at vt): p as kTerms terms of B fragments,
// in the order of the keys that scores32 leaves.
template <int DH, bool F16>
__device__ __forceinline__ void values16(const uint8_t* vt, const uint32_t (&t)[4][kTerms], floatx16 (&o)[DH / 32],
                                         int lane = threadIdx.x & 63) {
    const int i = lane & 15;
    const uint8_t* const row = vt + ((lane >> 5) * 4 + (i >> 2)) * (2 * DH) + ((lane >> 4) & 1) * 32 + (i & 3) * 8;
    const int x = perm_v<DH>(i >> 2) / 4;
#pragma unroll
    for (int d = 0; d < DH / 32; d++) {
        const uint2 lo = lds_read_tr(row + (d ^ x) * 64), hi = lds_read_tr(row + (d ^ x) * 64 + 16 * DH);
        const uint4 vf = make_uint4(lo.x, lo.y, hi.x, hi.y);
#pragma unroll
        for (int n = kTerms - 1; n >= 0; n--) o[d] = mfma<F16>(vf, make_uint4(t[0][n], t[1][n], t[2][n], t[3][n]), o[d]);
    }
}

// One tile of 32 * N keys (from k0) of the online softmax: scores to weights in place.
// sees(k): with TREE, of the 32 keys from k on those that the lane's row sees.
template <int DH, bool F16, bool TREE, int N, class Sees>
__device__ __forceinline__ float mask_and_move(floatx16 (&s)[N], int k0, int lim, bool edge, Sees sees, float c, float& m, float& l,
                                               floatx16 (&o)[DH / 32], int lane = threadIdx.x & 63) {
    const int h = lane >> 5;
    // register r of s[g] is key k0 + 32 g + 8 (r / 4) + 4 h + r % 4
    if constexpr (TREE) {
        if (edge)
#pragma unroll
            for (int g = 0; g < N; g++) {
                const uint32_t bits = sees(k0 + 32 * g) >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (!(bits & (1u << (8 * (r >> 2) + (r & 3))))) s[g][r] = ninf();
            }
    } else if (edge) {
#pragma unroll
        for (int g = 0; g < N; g++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (k0 + 32 * g + 8 * (r >> 2) + 4 * h + (r & 3) >= lim) s[g][r] = ninf();
    }
    float mt = ninf();
#pragma unroll
    for (int g = 0; g < N; g++)
#pragma unroll
        for (int r = 0; r < 16; r++) mt = fmaxf(mt, s[g][r]);
    mt = pair32<true>(mt) * c;
    if (__any(mt > m + kLazy<F16>)) {
        const float mn = fmaxf(m, mt);
        const float f = mn == ninf() ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
#pragma unroll
        for (int d = 0; d < DH / 32; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] *= f;
        m = mn;
    }
    return m == ninf() ? 0.0f : kPShift<F16> - m;
}
// (neg: mask_and_move's)
template <int N>
__device__ __forceinline__ void weigh(floatx16 (&s)[N], float c, float neg, float& l) {
    float sum = 0.0f;
#pragma unroll
    for (int g = 0; g < N; g++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            s[g][r] = __builtin_amdgcn_exp2f(fmaf(s[g][r], c, neg));
            sum += s[g][r];
        }
    l += sum;
}

// Products and exponentials use different units, but only as far as their instructions
// alternate; the order here is the source's (sched_barrier), with operands read two products ahead.
// Left to the compiler, all products came first: a tree of 63 tokens (252 rows, head_dim 128) over
// 30000 keys took 62 us for its parts instead of 58; 64 trees of 32 tokens over 4000 keys of head_dim
// 64 took 163 us instead of 147.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// scores32 of a tile of 32 N keys into `next`, and weigh of the tile before it.
template <int DH, bool F16, int N>
__device__ __forceinline__ void scores_and_weigh(const uint8_t* kt, const uint4 (&qf)[DH / 16], floatx16 (&next)[N],
                                                 floatx16 (&s)[N], float c, float neg, float& l, int lane) {
    constexpr int kSteps = N * DH / 16, kEach = 16 * N / kSteps;
    const int row = lane & 31, x = ((lane >> 5) ^ perm_k<DH>(row)) * 16;
    const uint8_t* const at = kt + row * (2 * DH);
    auto key = [&](int i) { return lds_read16(at + (i % N) * 64 * DH + (x ^ (32 * (i / N)))); };
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int r = 0; r < 16; r++) next[n][r] = 0.0f;
    uint4 k[3] = {key(0), key(1), key(0)};
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
        if (i + 2 < kSteps) k[(i + 2) % 3] = key(i + 2);
        next[i % N] = mfma<F16>(k[i % 3], qf[i / N], next[i % N]);
#pragma unroll
        for (int e = i * kEach; e < (i + 1) * kEach; e++) {
            s[e >> 4][e & 15] = __builtin_amdgcn_exp2f(fmaf(s[e >> 4][e & 15], c, neg));
            sum += s[e >> 4][e & 15];
        }
        in_order();
    }
    l += sum;
}
// values16 over 32 N keys.
template <int DH, bool F16, int N>
__device__ __forceinline__ void values(const uint8_t* vt, const floatx16 (&s)[N], floatx16 (&o)[DH / 32], int lane) {
    constexpr int kD = DH / 32, kSteps = 2 * N * kD;
    const int i16 = lane & 15, x = perm_v<DH>(i16 >> 2) / 4;
    const uint8_t* const at = vt + ((lane >> 5) * 4 + (i16 >> 2)) * (2 * DH) + ((lane >> 4) & 1) * 32 + (i16 & 3) * 8;
    auto value = [&](int i) {
        const uint8_t* const p = at + (i / kD) * 32 * DH + ((i % kD) ^ x) * 64;
        const uint2 lo = lds_read_tr(p), hi = lds_read_tr(p + 16 * DH);
        return make_uint4(lo.x, lo.y, hi.x, hi.y);
    };
    uint32_t p[2][4][kTerms];
    auto split = [&](int kk, int e) {
        split_pair<F16, kTerms>(s[kk >> 1][8 * (kk & 1) + 2 * e], s[kk >> 1][8 * (kk & 1) + 2 * e + 1], p[kk & 1][e]);
    };
    uint4 v[2] = {value(0), value(0)};
#pragma unroll
    for (int e = 0; e < 4; e++) split(0, e);
    in_order();
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
        const int kk = i / kD, d = i % kD;
        if (i + 1 < kSteps) v[(i + 1) & 1] = value(i + 1);
#pragma unroll
        for (int n = kTerms - 1; n >= 0; n--)
            o[d] = mfma<F16>(v[i & 1], make_uint4(p[kk & 1][0][n], p[kk & 1][1][n], p[kk & 1][2][n], p[kk & 1][3][n]), o[d]);
        if (kk + 1 < 2 * N)
#pragma unroll
            for (int e = d * 4 / kD; e < (d + 1) * 4 / kD; e++) split(kk + 1, e);
        in_order();
    }
}

// The wave's rows (bit lane % 32) whose results are not finite.
template <int DH>
__device__ __forceinline__ uint32_t rows_again(float l, const floatx16 (&o)[DH / 32], bool live) {
    float z = l * 0.0f;  // NaN once something is not finite
#pragma unroll
    for (int d = 0; d < DH / 32; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) z = fmaf(o[d][r], 0.0f, z);
    const uint64_t votes = __ballot(z != z && live);
    return (uint32_t)votes | (uint32_t)(votes >> 32);
}

__device__ __forceinline__ int wave_min_int(int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = min(v, __shfl_xor(v, d, 64));
    return v;
}

}  // namespace
}  // namespace jh
