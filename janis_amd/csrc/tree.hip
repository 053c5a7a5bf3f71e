// Trees of drafted tokens over the paged cache: positions and masks, the path that the
// model agrees with, and its keys and values moved together (attention:
// paged_attention.hip).
#include "jh_common.hpp"

namespace jh {
namespace {

// The lanes of a wave see each other's LDS stores.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---- positions and masks -----------------------------------------------------------
// A wave to a request, 64 rows at a time, a lane to a row. Within the 64, ancestors are
// found by doubling: each round a lane takes over the bits of the row that it points to
// and points where that one does, so a way up of d rows takes log2 d rounds of lane
// exchanges and no memory. A way that leaves the 64 goes on at a row whose mask is
// there already (in LDS). Depth is the number of bits. Blocks past the requests look
// after the rows that belong to nobody.
constexpr int kFillThreads = 64;
template <int W>  // mask words, or 0: any number
__global__ __launch_bounds__(64) void tree_plan_kernel(TreePlanArgs a) {
    extern __shared__ uint32_t s_mask[];  // [32 words][words], where a request may have more than 64 rows
    const int words = W ? W : a.words, lane = threadIdx.x, r = blockIdx.x;
    auto put = [&](int t, int position) {
        a.positions[t] = position;
    };
    if (r >= a.n_req) {
        const int first = a.n_req ? min(max(a.row_starts[0], 0), a.n_rows) : a.n_rows;
        const int last = a.n_req ? min(max(a.row_starts[a.n_req], first), a.n_rows) : a.n_rows;
        const int nobodys = first + a.n_rows - last;
        for (int i = (r - a.n_req) * kFillThreads + lane; i < nobodys; i += (gridDim.x - a.n_req) * kFillThreads) {
            const int t = i < first ? i : i - first + last;
            put(t, -1);
            for (int w = 0; w < words; w++) a.mask[(int64_t)t * words + w] = 0;
        }
        return;
    }
    const int from = a.row_starts[r], to = a.row_starts[r + 1], kv = a.kv_lens[r];
    const int start = min(max(from, 0), a.n_rows), n = min(max(to, start), a.n_rows) - start;
    const int base = kv - n;
    if (n > 32 * words) {
        for (int i = lane; i < n; i += 64) {
            put(start + i, base + i);
            for (int w = 0; w < words; w++) a.mask[(int64_t)(start + i) * words + w] = 0;
        }
        return;
    }
    for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        int p = i < n ? a.parents[start + i] : -1;
        if (p < -1 || p >= i) p = -1;
        uint64_t bits = 1ull << lane;
        int up = p >= i0 ? p - i0 : -1;     // lane that the way up has come to, -1: it has left the 64
        int out = p >= i0 ? -1 : p;         // then, the earlier row that it goes on at
        while (__any(up >= 0)) {
            const int at = max(up, 0);
            const uint64_t more = (uint64_t)(uint32_t)__shfl((int)(bits >> 32), at, 64) << 32 | (uint32_t)__shfl((int)bits, at, 64);
            const int next = __shfl(up, at, 64), leaves = __shfl(out, at, 64);
            if (up >= 0) {
                bits |= more;
                up = next;
                if (next < 0) out = leaves;
            }
        }
        int depth = __popcll(bits) - 1;
        if (i < n) {
            for (int w = 0; w < words; w++) {
                uint32_t v = 0;
                const int part = w - i0 / 32;
                if (part >= 0) {
                    v = part == 0 ? (uint32_t)bits : part == 1 ? (uint32_t)(bits >> 32) : 0u;
                } else if (out >= 0) {
                    v = s_mask[out * words + w];
                    depth += __popc(v);
                }
                a.mask[(int64_t)(start + i) * words + w] = v;
                if (n > 64) s_mask[i * words + w] = v;
            }
            put(start + i, base + depth);
        }
        if (n > 64) wave_fence();
    }
}

// ---- the path that the model agrees with ----------------------------------------------
// One workgroup: lengths and the stack are updated in place, so all that decides is read
// before the barrier behind which anything is written. Rows (parents, tokens, choices)
// come to LDS kRows at a time, all requested together; a thread walks its requests
// there in one pass, since a child comes after its parent: row i is kept if its parent
// is the last row kept and its token the choice there.
constexpr int kCommitThreads = 1024, kRows = 8192;
static_assert(kPlanMaxReq % kCommitThreads == 0, "requests per thread");

__device__ __forceinline__ int scan_int(int v) {  // sum over the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d, 64);
        if ((int)(threadIdx.x & 63) >= d) v += u;
    }
    return v;
}

__global__ __launch_bounds__(kCommitThreads) void tree_commit_kernel(TreeCommitArgs a) {
    constexpr int kPer = kPlanMaxReq / kCommitThreads, kWaves = kCommitThreads / 64;
    __shared__ int s_parent[kRows], s_token[kRows], s_chosen[kRows];
    __shared__ int s_start[kPlanMaxReq + 1], s_kept[kPlanMaxReq];  // (~kept: of a run, kept whole)
    __shared__ int s_known[kPlanMaxReq];
    __shared__ int s_sum[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, R = a.n_req, page = 1 << a.page_shift;
    const int64_t limit = min((int64_t)a.max_blocks << a.page_shift, (int64_t)0x7fffffff);
    auto blocks = [&](int64_t kv) { return (int)((kv + page - 1) >> a.page_shift); };
    const int count = *a.free_count;
    int start[kPer], n[kPer], kv[kPer], known[kPer];
    bool lengths = false, rows = false;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int r = tid * kPer + e;
        start[e] = n[e] = kv[e] = known[e] = 0;
        if (r >= R) continue;
        start[e] = a.row_starts[r];
        const int to = a.row_starts[r + 1];
        kv[e] = a.kv_lens[r];
        const bool wrong = start[e] < 0 || to < start[e] || to > a.n_rows;
        rows |= wrong;
        n[e] = wrong ? 0 : to - start[e];
        lengths |= kv[e] < n[e] || kv[e] > limit;
        known[e] = n[e] > a.tree_rows ? n[e] : min(max(a.known ? a.known[r] : 1, 1), n[e]);
        s_start[r] = start[e];
        s_known[r] = known[e];
    }
    if (tid == 0 && R > 0) s_start[R] = a.row_starts[R];
    lengths = __syncthreads_or(lengths);
    rows = __syncthreads_or(rows);
    int status = lengths ? JH_PLAN_LENGTHS : rows ? JH_PLAN_ROWS : count < 0 || count > a.n_pages ? JH_PLAN_PAGES : JH_PLAN_OK;
    int at[kPer], cur[kPer], want[kPer], kept[kPer];
#pragma unroll
    for (int e = 0; e < kPer; e++) at[e] = known[e] - 1, cur[e] = -1, want[e] = -1, kept[e] = known[e];
    const int first = status == JH_PLAN_OK && R > 0 ? s_start[0] : 0, last = status == JH_PLAN_OK && R > 0 ? s_start[R] : 0;
    for (int w0 = first; w0 < last; w0 += kRows) {
        const int w1 = min(last, w0 + kRows);
        if (w0 > first) __syncthreads();  // (the walks before have read)
#pragma unroll
        for (int e = 0; e < kRows / kCommitThreads; e++) {
            const int t = w0 + e * kCommitThreads + tid;
            if (t >= w1) continue;
            s_parent[t - w0] = a.parents[t];
            s_token[t - w0] = a.tokens[t];
            s_chosen[t - w0] = a.chosen[t * a.chosen_stride];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            if (n[e] == 0) continue;
            const int end = min(n[e], w1 - start[e]);
            for (; at[e] < end; at[e]++) {
                const int i = at[e], x = start[e] + i - w0;
                if (i == known[e] - 1) {
                    cur[e] = i, want[e] = s_chosen[x];
                } else if (s_parent[x] == cur[e] && s_token[x] == want[e]) {
                    a.path[start[e] + kept[e]] = start[e] + i;
                    cur[e] = i, want[e] = s_chosen[x];
                    kept[e]++;
                }
            }
        }
    }
    // pages that come back: a request's lie behind those of the requests before it
    int back[kPer], run = 0;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        back[e] = status == JH_PLAN_OK ? blocks(kv[e]) - blocks(kv[e] - n[e] + kept[e]) : 0;
        run += back[e];
    }
    const int upto = scan_int(run);
    if (lane == 63) s_sum[wave] = upto;
    bool outside = false;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int r = tid * kPer + e;
        const int b = blocks(kv[e] - n[e] + kept[e]);
        for (int j = 0; j < back[e]; j++) outside |= (uint32_t)a.tables[(int64_t)r * a.max_blocks + b + j] >= (uint32_t)a.n_pages;
    }
    outside = __syncthreads_or(outside);
    int total = 0, to = count + upto - run;
    for (int w = 0; w < kWaves; w++) {
        if (w < wave) to += s_sum[w];
        total += s_sum[w];
    }
    if (status == JH_PLAN_OK && (outside || (int64_t)count + total > a.n_pages)) status = JH_PLAN_TABLE;
    const bool ok = status == JH_PLAN_OK;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int r = tid * kPer + e;
        if (r >= R) continue;
        const int left = kv[e] - n[e] + kept[e];
        a.kv_out[r] = ok ? left : kv[e];
        a.accepted[r] = ok ? kept[e] : 0;
        a.next_tokens[r] = ok ? want[e] : -1;
        s_kept[r] = kept[e];
        if (ok)
            for (int j = 0; j < back[e]; j++) a.free_pages[to++] = a.tables[(int64_t)r * a.max_blocks + blocks(left) + j];
    }
    if (tid == 0) {
        *a.status = status;
        *a.count_out = ok ? count + total : count;
    }
    if (!ok) {
        for (int t = tid; t < a.n_rows; t += kCommitThreads) a.path[t] = -1;
        return;
    }
    __syncthreads();
    // the known rows' places, and those that no row has
    for (int t = tid; t < a.n_rows; t += kCommitThreads) {
        int v = -1;
        if (t >= first && t < last) {
            int lo = 0;
            for (int len = R; len > 1;) {  // the last request that starts at or before t
                const int half = len >> 1;
                if (s_start[lo + half] <= t) lo += half;
                len -= half;
            }
            const int i = t - s_start[lo];
            if (i < s_known[lo]) v = t;
            else if (i < s_kept[lo]) continue;  // (written by the walk)
        }
        a.path[t] = v;
    }
}

// ---- keys and values of the path moved together ------------------------------------------
// A block to a request and layer, a thread to 16 bytes of a key's or value's heads. Row j
// of the path moves to slot j of the request, j <= path[j]: kTogether rows are read
// before they are written, and what later rows read lies behind what is written.
constexpr int kTogether = 8;
__global__ __launch_bounds__(256) void tree_move_kernel(TreeMoveArgs a) {
    const int r = blockIdx.x, layer = blockIdx.y, lane = threadIdx.x & 63;
    const int start = a.row_starts[r], kept = a.accepted[r];
    if (kept <= 0 || start < 0 || start > a.n_rows - kept) return;
    const int32_t* const path = a.path + start;
    if (path[kept - 1] == start + kept - 1) return;  // all are where they belong
    const int pieces = a.Dh / 8, per = a.Hk * pieces;
    for (int j0 = 0; j0 < kept; j0 += 64) {
        // the lanes look up 64 rows
        const int j = j0 + lane, from = j < kept ? path[j] : -1;
        int src = -1, dst = -1;
        if (from >= 0 && from < a.n_rows && from != start + j) src = a.slots[from], dst = a.slots[start + j];
        const uint64_t moves = __ballot((uint32_t)src < (uint32_t)a.n_slots && (uint32_t)dst < (uint32_t)a.n_slots);
        for (int i = threadIdx.x; i < 2 * per; i += 256) {
            uint16_t* const pool = i < per ? a.k[layer] : a.v[layer];
            const int x = i < per ? i : i - per, head = x / pieces, f = 8 * (x % pieces);
            auto where = [&](int slot) {
                const int row = slot & ((1 << a.page_shift) - 1);
                return reinterpret_cast<uint4*>(pool + (slot >> a.page_shift) * a.page_stride +
                                                (((int64_t)head << a.page_shift) + row) * a.Dh + f);
            };
            uint64_t left = moves;
            while (left) {
                uint4 v[kTogether];
                int to[kTogether];
#pragma unroll
                for (int e = 0; e < kTogether; e++) {
                    to[e] = -1;
                    if (!left) continue;
                    const int l = __ffsll((unsigned long long)left) - 1;
                    left &= left - 1;
                    v[e] = *where(__builtin_amdgcn_readlane(src, l));
                    to[e] = __builtin_amdgcn_readlane(dst, l);
                }
#pragma unroll
                for (int e = 0; e < kTogether; e++)
                    if (to[e] >= 0) *where(to[e]) = v[e];
            }
        }
    }
}

}  // namespace

Status launch_tree_plan(const TreePlanArgs& a, hipStream_t st) {
    const unsigned fill = (unsigned)std::min<int64_t>(64, ((int64_t)a.n_rows + kFillThreads - 1) / kFillThreads);
    const dim3 grid((unsigned)a.n_req + fill);
    // requests of more than 64 rows keep their masks in LDS: up to 32 KB
    if (a.words == 1) hipLaunchKernelGGL(tree_plan_kernel<1>, grid, dim3(64), 0, st, a);
    else if (a.words == 2) hipLaunchKernelGGL(tree_plan_kernel<2>, grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL(tree_plan_kernel<0>, grid, dim3(64), (size_t)128 * a.words * a.words, st, a);
    return Status::ok();
}

Status launch_tree_commit(const TreeCommitArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(tree_commit_kernel, dim3(1), dim3(kCommitThreads), 0, st, a);
    return Status::ok();
}

Status launch_tree_move(const TreeMoveArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(tree_move_kernel, dim3((unsigned)a.n_req, (unsigned)a.layers), dim3(256), 0, st, a);
    return Status::ok();
}

}  // namespace jh
