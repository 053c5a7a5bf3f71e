// A paged key/value cache for batches of requests: the bookkeeping of a step and
// the append of new rows (attention over the pages: paged_attention.hip).
#include "jh_common.hpp"

namespace jh {
namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// ---- bookkeeping ---------------------------------------------------------------
// One workgroup: what it reads may be what it writes (lengths and the stack are
// updated in place), so everything that decides is read before the barrier behind which
// anything is written; what is read later (the stack below *free_count, finished
// requests' tables, the last page of the others) is never written here. Requests' new
// rows, new pages and pages that come back are running sums in LDS (one scan of up to
// 2048 requests over 1024 threads), and a row or page finds its request by bisection,
// kTogether of them to a thread at once. Bound: latency -- the lengths' round trip, the
// scan's barriers, the pages' round trip, the tables' and the stores. MI355X: 64 requests
// of one new token 5.7 us, 700 requests with 8192 rows 14.6 us, of which 0.15 and 0.5 are
// the look at the pages that requests go on filling. Without it 14.1, where one row or page
// to a thread at a time took 16.0, two 14.4 and eight 13.9 (64 requests then 1 us more).
constexpr int kPlanThreads = 1024, kTogether = 4;
static_assert(kPlanMaxReq % kPlanThreads == 0, "requests per thread");

// The last i of 0 .. n - 1 with v[i] <= x (v never decreases, v[0] <= x).
__device__ __forceinline__ int owner_of(const int* v, int n, int x) {
    int lo = 0;
    while (n > 1) {
        const int half = n >> 1;
        if (v[lo + half] <= x) lo += half;
        n -= half;
    }
    return lo;
}

template <bool ROW>
__device__ __forceinline__ int scan_int(int v) {  // sum over the lanes up to this one (ROW: of its 16)
    auto dpp = [](int x, auto ctrl, auto rows) {
        return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    };
    using All = std::integral_constant<int, 0xF>;
    v += dpp(v, std::integral_constant<int, 0x111>{}, All{});  // row_shr:1
    v += dpp(v, std::integral_constant<int, 0x112>{}, All{});  // row_shr:2
    v += dpp(v, std::integral_constant<int, 0x114>{}, All{});  // row_shr:4
    v += dpp(v, std::integral_constant<int, 0x118>{}, All{});  // row_shr:8
    if constexpr (!ROW) {
        v += dpp(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row_bcast:15
        v += dpp(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row_bcast:31
    }
    return v;
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedPlanArgs a, int shift) {
    constexpr int kPer = kPlanMaxReq / kPlanThreads, kWaves = kPlanThreads / 64;
    static_assert(kWaves == 16, "the waves' sums are one row of lanes");
    // running sums over the requests before each; keys held before (~keys: finished)
    __shared__ int s_row[kPlanMaxReq], s_take[kPlanMaxReq], s_back[kPlanMaxReq], s_kv[kPlanMaxReq];
    __shared__ int s_sum[3][kWaves];
    __shared__ float s_about[3][kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, R = a.n_req;
    const int64_t limit = min((int64_t)a.max_blocks << shift, (int64_t)0x7fffffff);
    const int count = *a.free_count;
    auto blocks = [&](int64_t kv) { return (int)((kv + a.page_size - 1) >> shift); };
    int kv[kPer], n[kPer], add[kPer][3];
    int run[3] = {0, 0, 0};           // rows, pages to take, pages that come back
    float about[3] = {0.0f, 0.0f, 0.0f};  // the same, where 32 bits may not hold them
    bool bad = false, out = false;  // out: a page number that is used lies outside the pool
    int last[kPer];
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int r = tid * kPer + e;
        kv[e] = r < R ? a.kv_lens[r] : 0;
        n[e] = r < R ? a.new_lens[r] : 0;
    }
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const bool wrong = kv[e] < 0 || kv[e] > limit || (int64_t)kv[e] + max(n[e], 0) > limit;
        bad |= wrong;
        const int held = wrong ? 0 : blocks(kv[e]);
        // new tokens that begin inside the last page held: its number is on its way beside the scan
        last[e] = !wrong && n[e] > 0 && (kv[e] & (a.page_size - 1))
                      ? a.tables[(int64_t)(tid * kPer + e) * a.max_blocks + held - 1] : 0;
        add[e][0] = wrong ? 0 : max(n[e], 0);
        add[e][1] = wrong || n[e] < 0 ? 0 : blocks((int64_t)kv[e] + n[e]) - held;
        add[e][2] = n[e] < 0 ? held : 0;
#pragma unroll
        for (int c = 0; c < 3; c++) run[c] += add[e][c], about[c] += (float)add[e][c];
    }
#pragma unroll
    for (int c = 0; c < 3; c++) {
        const int upto = scan_int<false>(run[c]);
        const float all = wave_sum(about[c]);
        if (lane == 63) s_sum[c][wave] = upto, s_about[c][wave] = all;
        run[c] = upto - run[c];
    }
    bad = __syncthreads_or(bad);
    int total[3];
#pragma unroll
    for (int c = 0; c < 3; c++) {
        const int upto = scan_int<true>(s_sum[c][lane & 15]);
        run[c] += wave ? __builtin_amdgcn_readlane(upto, wave - 1) : 0;
        total[c] = __builtin_amdgcn_readlane(upto, 15);
        about[c] = row16_sum(s_about[c][lane & 15]);
    }
    // sums past 1.5e9 are more than there can be (n_rows, n_pages: at most 2^30) ...
    const bool rows_over = about[0] > 1.5e9f, take_over = about[1] > 1.5e9f, back_over = about[2] > 1.5e9f;
    // ... and the others are exact
    const int64_t top = (int64_t)count + total[2];
    int status = JH_PLAN_OK;
    if (bad) status = JH_PLAN_LENGTHS;
    else if (rows_over || total[0] > a.n_rows) status = JH_PLAN_ROWS;
    else if (count < 0 || count > a.n_pages || (back_over ? about[1] > about[2] : take_over || total[1] > top))
        status = JH_PLAN_PAGES;
    else if (back_over || top > a.n_pages) status = JH_PLAN_TABLE;
    const int n_rows = total[0], n_take = total[1], n_back = total[2], n_most = max(n_take, n_back);
    // the number of page `k` of those that come back, and of those that come off the stack
    auto back_of = [&](int k) {
        const int r = owner_of(s_back, R, k);
        return a.tables[(int64_t)r * a.max_blocks + k - s_back[r]];
    };
    auto take_of = [&](int k) {
        const int at = (int)top - 1 - k;
        return at < count ? a.free_pages[at] : back_of(at - count);
    };
    int back[kTogether], take[kTogether];
    if (status == JH_PLAN_OK) {
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const int r = tid * kPer + e;
            s_row[r] = run[0], s_take[r] = run[1], s_back[r] = run[2];
            s_kv[r] = n[e] < 0 ? ~kv[e] : kv[e];
#pragma unroll
            for (int c = 0; c < 3; c++) run[c] += add[e][c];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kPer; e++) out |= (uint32_t)last[e] >= (uint32_t)a.n_pages && n[e] > 0;
#pragma unroll
        for (int e = 0; e < kTogether; e++) {
            const int k = tid + e * kPlanThreads;
            if (e * kPlanThreads >= n_most) break;
            back[e] = k < n_back ? back_of(k) : 0;
            take[e] = k < n_take ? take_of(k) : 0;
            out |= (uint32_t)back[e] >= (uint32_t)a.n_pages && k < n_back;
            out |= (uint32_t)take[e] >= (uint32_t)a.n_pages && k < n_take;
        }
        for (int k = tid + kTogether * kPlanThreads; k < n_most; k += kPlanThreads) {
            if (k < n_back) out |= (uint32_t)back_of(k) >= (uint32_t)a.n_pages;
            if (k < n_take) out |= (uint32_t)take_of(k) >= (uint32_t)a.n_pages;
        }
        if (__syncthreads_or(out)) status = JH_PLAN_TABLE;
    }
    const bool ok = status == JH_PLAN_OK;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int r = tid * kPer + e;
        if (r >= R) continue;
        a.kv_out[r] = !ok ? kv[e] : n[e] < 0 ? 0 : kv[e] + n[e];
        a.row_starts[r] = ok ? s_row[r] : 0;
    }
    if (tid == 0) {
        *a.status = status;
        *a.count_out = ok ? (int)top - n_take : count;
        a.row_starts[R] = ok ? n_rows : 0;
    }
    if (!ok) {
        for (int i = tid; i < a.n_rows; i += kPlanThreads) a.positions[i] = a.slots[i] = -1;
        return;
    }
    auto put_taken = [&](int k, int page) {
        const int r = owner_of(s_take, R, k);
        a.tables[(int64_t)r * a.max_blocks + blocks(s_kv[r]) + k - s_take[r]] = page;
    };
#pragma unroll
    for (int e = 0; e < kTogether; e++) {
        const int k = tid + e * kPlanThreads;
        if (e * kPlanThreads >= n_most) break;
        if (k < n_back) a.free_pages[count + k] = back[e];
        if (k < n_take) put_taken(k, take[e]);
    }
    for (int k = tid + kTogether * kPlanThreads; k < n_most; k += kPlanThreads) {
        if (k < n_back) a.free_pages[count + k] = back_of(k);
        if (k < n_take) put_taken(k, take_of(k));
    }
    for (int first = 0; first < a.n_rows; first += kTogether * kPlanThreads) {
        int pos[kTogether], page[kTogether];
#pragma unroll
        for (int e = 0; e < kTogether; e++) {
            const int i = first + e * kPlanThreads + tid;
            if (i - tid >= a.n_rows) break;
            pos[e] = page[e] = -1;
            if (i >= n_rows) continue;
            const int r = owner_of(s_row, R, i), held = blocks(s_kv[r]);
            pos[e] = s_kv[r] + i - s_row[r];
            const int b = pos[e] >> shift;
            page[e] = b < held ? a.tables[(int64_t)r * a.max_blocks + b] : take_of(s_take[r] + b - held);
        }
#pragma unroll
        for (int e = 0; e < kTogether; e++) {
            const int i = first + e * kPlanThreads + tid;
            if (i >= a.n_rows) break;
            a.positions[i] = pos[e];
            a.slots[i] = pos[e] >= 0 ? (page[e] << shift) + (pos[e] & (a.page_size - 1)) : -1;
        }
    }
}

// ---- append ---------------------------------------------------------------------
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2_t f = {a, b};
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, f16x2_t));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2_t));
}

// x of the lane LANES / 2 away in its group of LANES, and the group's sum, in every lane.
template <int LANES>
__device__ __forceinline__ float other_half(float x) {
    if constexpr (LANES == 16)
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xF, 0xF,
                                                                     false));  // row_ror:8
    return __shfl_xor(x, LANES / 2, 64);
}
template <int LANES>
__device__ __forceinline__ float group_sum(float x) {
    if constexpr (LANES >= 16) {
        x = row16_sum(x);
        return LANES == 32 ? pair16<false>(x) : x;
    }
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) x += __shfl_xor(x, d, 64);
    return x;
}

// A wave takes heads of one row, 64 / (DH / 8) of them at a time with 8 features per
// lane; the feature that is rotated with one lies half a head away, DH / 16 lanes on.
// kAhead times that many heads are requested together, the first before anything else;
// while they are on their way the lanes evaluate the rotation's factors, a pair each:
// the angle in double, its whole turns taken off there, sine and cosine of the rest in
// fp32 (within 2^-23). Calls of few rows share a row's heads among `share` waves.
// Bound: many rows, HBM; few, the round trips of slot, position and row. MI355X, 32 and 8
// heads of 128: 1 bf16 row 3.2 us, 4001 rows 22 us (98 MB, 4.4 TB/s; a block to a row
// took 35 us). kAhead: one 3.1 and 23.9 us, three 3.6 and 22.6; at 8000 rows one
// loses 4 us.
constexpr int kAhead = 2;
template <int DH, bool F16, bool F32>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, int share) {
    constexpr int kLanes = DH / 8, kHeads = 64 / kLanes, kHalf = DH / 2;
    __shared__ float2 s_turn[4][kHalf];
    const int lane = threadIdx.x & 63, l = lane % kLanes, heads = a.Hq + 2 * a.Hk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int t = (int)(item / share), step = share * kHeads;
    if (t >= a.n_rows) return;
    const int slot = a.slots[t];
    const bool turn = a.freqs || a.base != 0.0f;
    const int pos = turn ? a.positions[t] : 0;
    const char* const from = static_cast<const char*>(a.qkv) + ((int64_t)t * a.qkv_stride + 8 * l) * (F32 ? 4 : 2);
    uint4 in[kAhead][F32 ? 2 : 1];
    auto load = [&](int first) {
#pragma unroll
        for (int n = 0; n < kAhead; n++) {
            const int head = min(first + n * step, heads - 1);  // (past the last: it again)
            const uint4* const p = reinterpret_cast<const uint4*>(from + (int64_t)head * DH * (F32 ? 4 : 2));
            in[n][0] = p[0];
            if constexpr (F32) in[n][1] = p[1];
        }
    };
    int first = (int)(item % share) * kHeads + lane / kLanes;
    load(first);
    float c[8], sn[8], qw[8], kw[8];  // the lane's features' factors (sn: of the other half's) and weights
    auto weights = [&](const void* w, float (&v)[8]) {
        if (!w) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = 1.0f;
        } else if (a.w_dt == JH_F32) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = static_cast<const float*>(w)[8 * l + e];
        } else if (a.w_wide) {
            const uint4 u = static_cast<const uint4*>(w)[l];
            const uint32_t us[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint16_t h = (uint16_t)(e & 1 ? us[e / 2] >> 16 : us[e / 2]);
                v[e] = a.w_dt == JH_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = load_sb(w, 8 * l + e, a.w_dt);
        }
    };
    weights(a.qn_w, qw);
    weights(a.kn_w, kw);
    if ((uint32_t)slot >= (uint32_t)a.n_slots) return;
    if (turn) {
        for (int i = lane; i < kHalf; i += 64) {
            const double inv = a.freqs ? 1.0 / (double)a.freqs[i] : exp2((double)i * a.log2_step);
            const double turns = (double)pos * (double)a.scale * inv * 0.15915494309189533577;
            float s, co;
            sincospif(2.0f * (float)(turns - rint(turns)), &s, &co);
            s_turn[wave][i] = make_float2(co, s);
        }
        // (the lanes read each other's factors)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float2 f = turn ? s_turn[wave][(8 * l + e) % kHalf] : make_float2(1.0f, 0.0f);
        c[e] = f.x, sn[e] = l < kLanes / 2 ? -f.y : f.y;
    }
    const int page = slot >> a.page_shift, row = slot & ((1 << a.page_shift) - 1);
    const int64_t at = page * a.page_stride + (int64_t)row * DH + 8 * l;
    for (; first - lane / kLanes < heads; first += kAhead * step) {
#pragma unroll
        for (int n = 0; n < kAhead; n++) {
            const int head = first + n * step;
            if (head - lane / kLanes >= heads) break;  // (the wave's: the lanes exchange values)
            float x[8];
            const uint32_t u[4] = {in[n][0].x, in[n][0].y, in[n][0].z, in[n][0].w};
            if constexpr (F32) {
                const uint32_t v[4] = {in[n][1].x, in[n][1].y, in[n][1].z, in[n][1].w};
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = __uint_as_float(u[e]), x[4 + e] = __uint_as_float(v[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    x[2 * e] = __uint_as_float(u[e] << 16), x[2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u);
            }
            const bool is_q = head < a.Hq, is_v = head >= a.Hq + a.Hk;
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) ss = fmaf(x[e], x[e], ss);
            ss = group_sum<kLanes>(ss);
            const float inv = (is_q ? a.qn_w : a.kn_w) ? 1.0f / sqrtf(ss * (1.0f / DH) + a.eps) : 1.0f;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = x[e] * inv * (is_q ? qw[e] : kw[e]);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float z = other_half<kLanes>(y[e]);
                if (turn) y[e] = y[e] * c[e] + z * sn[e];
                if (is_v) y[e] = x[e];
            }
            if (head >= heads) continue;
            uint16_t* to;
            if (is_q) to = a.q_out + ((int64_t)t * a.Hq + head) * DH + 8 * l;
            else to = (is_v ? a.v : a.k) + at + ((int64_t)(head - a.Hq - (is_v ? a.Hk : 0)) << a.page_shift) * DH;
            *reinterpret_cast<uint4*>(to) = make_uint4(pack2<F16>(y[0], y[1]), pack2<F16>(y[2], y[3]),
                                                       pack2<F16>(y[4], y[5]), pack2<F16>(y[6], y[7]));
        }
        load(first + kAhead * step);
    }
}

}  // namespace

Status launch_paged_plan(const PagedPlanArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a, __builtin_ctz(a.page_size));
    return Status::ok();
}

Status launch_paged_append(const PagedAppendArgs& a, int num_cus, hipStream_t st) {
    // waves to a row: enough to give every SIMD four, at most one for each 64 * 8 features
    const int64_t all = ((int64_t)(a.Hq + 2 * a.Hk) * a.Dh + 511) / 512;
    const int share = (int)std::max<int64_t>(1, std::min(all, 16 * (int64_t)num_cus / a.n_rows));
    const dim3 grid((unsigned)(((int64_t)a.n_rows * share + 3) / 4));
    auto with = [&](auto dh, auto f16) {
        constexpr int DH = decltype(dh)::value;
        constexpr bool F16 = decltype(f16)::value;
        if (a.qkv_dt == JH_F32) hipLaunchKernelGGL((paged_append_kernel<DH, F16, true>), grid, dim3(256), 0, st, a, share);
        else hipLaunchKernelGGL((paged_append_kernel<DH, F16, false>), grid, dim3(256), 0, st, a, share);
    };
    auto typed = [&](auto dh) { a.kv_f16 ? with(dh, std::true_type{}) : with(dh, std::false_type{}); };
    if (a.Dh == 64) typed(std::integral_constant<int, 64>{});
    else if (a.Dh == 128) typed(std::integral_constant<int, 128>{});
    else typed(std::integral_constant<int, 256>{});
    return Status::ok();
}

}  // namespace jh
