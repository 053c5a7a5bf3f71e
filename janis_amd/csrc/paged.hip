// A paged key/value cache for batches of requests: the bookkeeping of a step and
// the append of new rows (attention over the pages: paged_attention.hip).
#include "jh_common.hpp"

namespace jh {
namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// ---- bookkeeping ---------------------------------------------------------------
// One workgroup: what it reads may be what it writes (lengths and the stack are
// updated in place), so everything is read before the barrier behind which it is
// written. Requests' new rows and pages are running sums (one scan of 2048
// requests over 1024 threads), kept in LDS; a new page or row then finds its
// request by bisection. Bound: latency -- the lengths' round trip, the scan's
// barriers, the table's or stack's round trip, the stores.
constexpr int kPlanThreads = 1024;
static_assert(kPlanMaxReq % kPlanThreads == 0, "requests per thread");

// The last of v[0..n] (never decreasing) that is at most x; v[0] <= x < v[n].
__device__ __forceinline__ int owner_of(const int* v, int n, int x) {
    int lo = 0;
    while (n > 1) {
        const int half = n >> 1;
        if (v[lo + half] <= x) lo += half;
        n -= half;
    }
    return lo;
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedPlanArgs a, int shift) {
    constexpr int kPer = kPlanMaxReq / kPlanThreads, kWaves = kPlanThreads / 64;
    // exclusive running sums over the requests; keys held before (~keys: finished)
    __shared__ int s_row[kPlanMaxReq + 1], s_take[kPlanMaxReq + 1], s_back[kPlanMaxReq + 1], s_kv[kPlanMaxReq];
    __shared__ int64_t s_sum[kWaves][3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, R = a.n_req;
    const int64_t limit = min((int64_t)a.max_blocks << shift, (int64_t)0x7fffffff);
    const int count = *a.free_count;
    auto blocks = [&](int64_t kv) { return (int)((kv + a.page_size - 1) >> shift); };
    int kv[kPer], n[kPer];
    int64_t sum[3] = {0, 0, 0};  // rows, pages to take, pages that come back
    bool bad = false;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int r = tid * kPer + e;
        kv[e] = r < R ? a.kv_lens[r] : 0;
        n[e] = r < R ? a.new_lens[r] : 0;
        if (kv[e] < 0 || kv[e] > limit || (int64_t)kv[e] + max(n[e], 0) > limit) {
            bad = true;
            continue;
        }
        sum[0] += max(n[e], 0);
        if (n[e] >= 0) sum[1] += blocks((int64_t)kv[e] + n[e]) - blocks(kv[e]);
        else sum[2] += blocks(kv[e]);
    }
    int64_t run[3];
#pragma unroll
    for (int c = 0; c < 3; c++) {
        int64_t v = sum[c];
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t up = __shfl_up(v, d, 64);
            if (lane >= d) v += up;
        }
        if (lane == 63) s_sum[wave][c] = v;
        run[c] = v - sum[c];
    }
    bad = __syncthreads_or(bad);
    int64_t total[3] = {0, 0, 0};
    for (int w = 0; w < kWaves; w++)
#pragma unroll
        for (int c = 0; c < 3; c++) {
            if (w == wave) run[c] += total[c];
            total[c] += s_sum[w][c];
        }
    const int64_t top = count + total[2];
    int status = bad                                                                 ? JH_PLAN_LENGTHS
                 : total[0] > a.n_rows                                               ? JH_PLAN_ROWS
                 : count < 0 || count > a.n_pages || total[1] > top                  ? JH_PLAN_PAGES
                 : top > a.n_pages                                                   ? JH_PLAN_TABLE
                                                                                     : JH_PLAN_OK;
    if (status == JH_PLAN_OK) {
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const int r = tid * kPer + e;
            s_row[r] = (int)run[0], s_take[r] = (int)run[1], s_back[r] = (int)run[2];
            s_kv[r] = n[e] < 0 ? ~kv[e] : kv[e];
            run[0] += max(n[e], 0);
            if (n[e] >= 0) run[1] += blocks((int64_t)kv[e] + n[e]) - blocks(kv[e]);
            else run[2] += blocks(kv[e]);
        }
        if (tid == kPlanThreads - 1) s_row[kPlanMaxReq] = (int)run[0], s_take[kPlanMaxReq] = (int)run[1];
        __syncthreads();
        // the numbers that would go onto the stack, and those that come off it
        bool out = false;
        if (total[2] > 0)
            for (int r = wave; r < R; r += kWaves)
                if (s_kv[r] < 0)
                    for (int j = lane; j < blocks(~s_kv[r]); j += 64)
                        out |= (uint32_t)a.tables[(int64_t)r * a.max_blocks + j] >= (uint32_t)a.n_pages;
        for (int64_t k = tid; k < total[1]; k += kPlanThreads)
            if (top - 1 - k < count) out |= (uint32_t)a.free_pages[top - 1 - k] >= (uint32_t)a.n_pages;
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
        *a.count_out = ok ? (int)(top - total[1]) : count;
        a.row_starts[R] = ok ? (int)total[0] : 0;
    }
    if (!ok) {
        for (int i = tid; i < a.n_rows; i += kPlanThreads) a.positions[i] = a.slots[i] = -1;
        return;
    }
    if (total[2] > 0) {
        for (int r = wave; r < R; r += kWaves)
            if (s_kv[r] < 0)
                for (int j = lane; j < blocks(~s_kv[r]); j += 64)
                    a.free_pages[count + s_back[r] + j] = a.tables[(int64_t)r * a.max_blocks + j];
        __threadfence_block();
        __syncthreads();
    }
    for (int k = tid; k < (int)total[1]; k += kPlanThreads) {
        const int r = owner_of(s_take, R, k);
        a.tables[(int64_t)r * a.max_blocks + blocks(s_kv[r]) + k - s_take[r]] = a.free_pages[top - 1 - k];
    }
    for (int i = tid; i < a.n_rows; i += kPlanThreads) {
        int pos = -1, slot = -1;
        if (i < (int)total[0]) {
            const int r = owner_of(s_row, R, i), held = blocks(s_kv[r]);
            pos = s_kv[r] + i - s_row[r];
            const int b = pos >> shift;
            const int page = b < held ? a.tables[(int64_t)r * a.max_blocks + b]
                                      : a.free_pages[top - 1 - (s_take[r] + b - held)];
            if ((uint32_t)page < (uint32_t)a.n_pages) slot = (page << shift) + (pos & (a.page_size - 1));
        }
        a.positions[i] = pos;
        a.slots[i] = slot;
    }
}

// ---- append ---------------------------------------------------------------------
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2_t f = {a, b};
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, f16x2_t));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2_t));
}

// A block takes heads of one row: 8 features per lane, DH / 8 lanes per head. The
// feature that is rotated with one lies half a head away, DH / 16 lanes on. The
// rotation's factors (double) are evaluated once per block, into LDS.
template <int DH, bool F16>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    constexpr int kLanes = DH / 8, kHeads = 256 / kLanes, kHalf = DH / 2;
    __shared__ float2 cs[kHalf];
    const int t = blockIdx.x, tid = threadIdx.x, l = tid % kLanes;
    const int slot = a.slots[t];
    if ((uint32_t)slot >= (uint32_t)a.n_slots) return;
    const bool turn = a.freqs || a.base != 0.0f;
    if (turn) {
        if (tid < kHalf) {
            const double inv = a.freqs ? 1.0 / (double)a.freqs[tid] : pow((double)a.base, (double)tid * (-2.0 / DH));
            double s, c;
            sincos((double)a.positions[t] * (double)a.scale * inv, &s, &c);
            cs[tid] = make_float2((float)c, (float)s);
        }
        __syncthreads();
    }
    const int heads = a.Hq + 2 * a.Hk;
    for (int head = blockIdx.y * kHeads + tid / kLanes; head < heads; head += gridDim.y * kHeads) {
        const int64_t at = (int64_t)t * a.qkv_stride + (int64_t)head * DH + 8 * l;
        float x[8];
        if (a.qkv_dt == JH_F32) {
            const float4* const p = reinterpret_cast<const float4*>(static_cast<const float*>(a.qkv) + at);
            const float4 u = p[0], v = p[1];
            x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.qkv) + at);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                x[2 * e] = __uint_as_float(w[e] << 16), x[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
        }
        const bool is_q = head < a.Hq, is_v = head >= a.Hq + a.Hk;
        const void* const w = is_v ? nullptr : is_q ? a.qn_w : a.kn_w;
        if (w) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) ss = fmaf(x[e], x[e], ss);
#pragma unroll
            for (int d = 1; d < kLanes; d <<= 1) ss += __shfl_xor(ss, d, 64);
            const float inv = 1.0f / sqrtf(ss * (1.0f / DH) + a.eps);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = x[e] * inv * load_sb(w, 8 * l + e, a.w_dt);
        }
        if (turn && !is_v) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = __shfl_xor(x[e], kLanes / 2, 64);
                const float2 f = cs[(8 * l + e) % kHalf];
                x[e] = x[e] * f.x + (l < kLanes / 2 ? -y : y) * f.y;
            }
        }
        const uint4 out = make_uint4(pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]), pack2<F16>(x[4], x[5]),
                                     pack2<F16>(x[6], x[7]));
        uint16_t* to;
        if (is_q) {
            to = a.q_out + ((int64_t)t * a.Hq + head) * DH;
        } else {
            const int h = head - a.Hq - (is_v ? a.Hk : 0);
            const int page = slot >> a.page_shift, row = slot & ((1 << a.page_shift) - 1);
            to = (is_v ? a.v : a.k) + page * a.page_stride + (((int64_t)h << a.page_shift) + row) * DH;
        }
        *reinterpret_cast<uint4*>(to + 8 * l) = out;
    }
}

}  // namespace

Status launch_paged_plan(const PagedPlanArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a, __builtin_ctz(a.page_size));
    return Status::ok();
}

Status launch_paged_append(const PagedAppendArgs& a, int num_cus, hipStream_t st) {
    const int passes = (a.Hq + 2 * a.Hk + 256 / (a.Dh / 8) - 1) / (256 / (a.Dh / 8));
    const dim3 grid((unsigned)a.n_rows, (unsigned)(a.n_rows < num_cus ? passes : 1));
    auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(256), 0, st, a); };
    if (a.kv_f16)
        a.Dh == 64    ? go(paged_append_kernel<64, true>)
        : a.Dh == 128 ? go(paged_append_kernel<128, true>)
                      : go(paged_append_kernel<256, true>);
    else
        a.Dh == 64    ? go(paged_append_kernel<64, false>)
        : a.Dh == 128 ? go(paged_append_kernel<128, false>)
                      : go(paged_append_kernel<256, false>);
    return Status::ok();
}

}  // namespace jh
