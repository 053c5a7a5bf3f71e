// Trees of drafted tokens over the paged cache: positions and masks, the path that the
// model agrees with, and its keys and values moved together (attention:
// paged_tree_attention.hip).
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
// after the rows that belong to nobody. Bound: two round trips; one request of 12 rows
// takes 1.5 us and 256 of 8 to 60 2.6, less than the host needs for a launch.
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
// Two launches: the first finds every request's path and what is to be done, in the
// workspace; the second does it. Nothing may be done if any request is wrong, lengths and
// the stack are updated in place, and what a request gives back lies on the stack behind
// what the ones before it give back: so all that decides comes before all that is written.
// Both are chains of round trips: two to the path (lengths; rows, their slots and the pages
// that may come back, all requested together), two to the writes (heads and moves; keys
// and values). With the walk and the books in one workgroup, and path and slots looked up
// by every block that moves, 64 requests of 8 to 32 rows in 36 layers took 33 us; so, 14.
// A single request that is not updated in place needs no more than itself: there every
// block of one launch finds the path (16 rows in 36 layers 6.7 us, with two launches 8.8).
//
// heads: per request {what is wrong with it or kFine, pages that come back, rows that move,
// its length}, behind them {*free_count}. moves: [request][most rows of a tree] of slots.
constexpr int kWalkThreads = 256, kTreeRows = 32 * JH_TREE_WORDS, kFine = 9;
static_assert(JH_PLAN_TABLE < kFine, "of several faults the least is reported");

// What a request's rows come to.
struct Walk {
    int4 head;       // as in heads
    int rows;
    int kept, next;  // rows kept, and the choice after the last
    int same;        // kept rows that stay where they are, the first ones
};
struct WalkRows {
    int parent[kTreeRows], token[kTreeRows], chosen[kTreeRows], slot[kTreeRows];
    int kept[kTreeRows];  // the kept rows
    int end[3];
};

// By all threads of a block. A child comes after its parent, so the path goes up: from row i
// on, the first row behind it whose parent is i and whose token the choice there, 64 rows to
// a ballot.
__device__ __forceinline__ Walk walk(const TreeCommitArgs& a, int r, WalkRows& s) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t limit = min((int64_t)a.max_blocks << a.page_shift, (int64_t)0x7fffffff);
    auto blocks = [&](int64_t kv) { return (int)((kv + (1 << a.page_shift) - 1) >> a.page_shift); };
    const int start = a.row_starts[r], to = a.row_starts[r + 1], kv = a.kv_lens[r];
    const int first = a.known ? a.known[r] : 1;
    const bool wrong = start < 0 || to < start || to > a.n_rows;
    const int n = wrong ? 0 : to - start;
    const int fault = kv < n || kv > limit ? JH_PLAN_LENGTHS : wrong ? JH_PLAN_ROWS : kFine;
    if (fault != kFine || n == 0) return Walk{make_int4(fault, 0, 0, kv), 0, 0, -1, 0};
    if (n > a.tree_rows) return Walk{make_int4(kFine, 0, 0, kv), n, n, a.chosen[(start + n - 1) * a.chosen_stride], n};
    const int known = min(max(first, 1), n), b0 = blocks(kv - n + known), back = blocks(kv) - b0;
    constexpr int kEach = kTreeRows / kWalkThreads;
    int page[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const int i = e * kWalkThreads + tid;
        page[e] = i < back ? a.tables[(int64_t)r * a.max_blocks + b0 + i] : 0;
        if (i >= n) continue;
        s.parent[i] = a.parents[start + i];
        s.token[i] = a.tokens[start + i];
        s.chosen[i] = a.chosen[(start + i) * a.chosen_stride];
        s.slot[i] = a.slots[start + i];
        s.kept[i] = i;
    }
    __syncthreads();
    if (tid < 64) {
        int at = known - 1, kept = known, same = known, want = s.chosen[at];
        for (int g = at >> 6; g < (n + 63) >> 6; g++) {
            const int i = min(64 * g + lane, n - 1);
            const int parent = s.parent[i], token = s.token[i], choice = s.chosen[i];
            for (;;) {
                const uint64_t next = __ballot(64 * g + lane < n && i > at && parent == at && token == want);
                if (!next) break;
                const int l = __ffsll((unsigned long long)next) - 1;
                at = 64 * g + l;
                want = __builtin_amdgcn_readlane(choice, l);
                same += at == kept;
                if (lane == 0) s.kept[kept] = at;
                kept++;
            }
        }
        if (lane == 0) s.end[0] = kept, s.end[1] = want, s.end[2] = same;
    }
    __syncthreads();
    const int kept = s.end[0], same = s.end[2], left = kv - n + kept, b = blocks(left) - b0;
    bool outside = false;
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const int i = e * kWalkThreads + tid;
        outside |= i >= b && i < back && (uint32_t)page[e] >= (uint32_t)a.n_pages;
    }
    outside = __syncthreads_or(outside);
    return Walk{make_int4(outside ? JH_PLAN_TABLE : kFine, back - b, kept - same, left), n, kept, s.end[1], same};
}

// The request's part of path, by all threads of a block.
__device__ __forceinline__ void write_path(const TreeCommitArgs& a, int r, const Walk& w, const WalkRows& s) {
    const int start = a.row_starts[r];
    for (int i = threadIdx.x; i < w.rows; i += kWalkThreads)
        a.path[start + i] = i >= w.kept ? -1 : start + (w.rows > a.tree_rows ? i : s.kept[i]);
}

// A block to a request.
__global__ __launch_bounds__(kWalkThreads) void tree_walk_kernel(TreeCommitArgs a) {
    __shared__ WalkRows s;
    const int r = blockIdx.x;
    if (r == 0 && threadIdx.x == 0) a.heads[a.n_req] = make_int4(*a.free_count, 0, 0, 0);
    const Walk w = walk(a, r, s);
    write_path(a, r, w, s);
    for (int i = threadIdx.x; i < w.head.z; i += kWalkThreads)
        a.moves[(int64_t)r * a.most + i] = make_int2(s.slot[s.kept[w.same + i]], s.slot[w.same + i]);
    if (threadIdx.x == 0) a.heads[r] = w.head, a.accepted[r] = w.kept, a.next_tokens[r] = w.next;
}

__device__ __forceinline__ int sum64(int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}
__device__ __forceinline__ int least64(int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = min(v, __shfl_xor(v, d, 64));
    return v;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Block (r, y): the books of request r (y 0, of the first launch), and its rows in the y-th part of
// the layers, a thread to 16 bytes of a key's or value's heads. The j-th kept row moves to slot j of
// the request, which is no kept row's behind it: so rows are read together, and written then. Every
// wave finds out for itself whether anything is done, while its first rows are on their way.
// ONE: a single request, whose path every block finds.
template <bool ONE>
__global__ __launch_bounds__(kWalkThreads) void tree_commit_kernel(TreeCommitArgs a, TreeMoveArgs m) {
    __shared__ typename std::conditional<ONE, WalkRows, int>::type s;
    const int r = blockIdx.x, R = a.n_req, tid = threadIdx.x, lane = tid & 63;
    const bool books = m.first && blockIdx.y == 0;
    const int l1 = min(m.layers, ((int)blockIdx.y + 1) * m.each);
    Walk w;
    if constexpr (ONE) w = walk(a, 0, s);
    int4 mine = ONE ? w.head : R ? a.heads[r] : make_int4(kFine, 0, 0, 0);
    if (m.layers == 0) mine.z = 0;
    if (!books && mine.z == 0) return;
    const int count = !ONE && R ? a.heads[R].x : *a.free_count;
    int2 head = make_int2(kFine, 0);
    if constexpr (ONE) head = make_int2(mine.x, lane == 0 ? mine.y : 0);
    else if (lane < R) head = make_int2(a.heads[lane].x, a.heads[lane].y);
    int status = -1, before = 0, total = 0;
    auto verdict = [&]() {
        int fault = head.x;
        total = head.y, before = lane < r ? head.y : 0;
        for (int i = lane + 64; !ONE && i < R; i += 64) {
            const int4 h = a.heads[i];
            fault = min(fault, h.x);
            total += h.y;
            if (i < r) before += h.y;
        }
        fault = least64(fault), total = sum64(total), before = sum64(before);
        if (count < 0 || count > a.n_pages) fault = min(fault, (int)JH_PLAN_PAGES);
        else if ((int64_t)count + total > a.n_pages) fault = min(fault, (int)JH_PLAN_TABLE);
        status = fault == kFine ? JH_PLAN_OK : fault;
    };
    const int pieces = m.Dh / 8, shift = __builtin_ctz(pieces | 1024), per = m.Hk * pieces;
    for (int j0 = 0; j0 < mine.z; j0 += 64) {
        const int count64 = min(64, mine.z - j0);
        const int mv = j0 + min(lane, count64 - 1);
        int2 slots;
        if constexpr (ONE) slots = make_int2(s.slot[s.kept[w.same + mv]], s.slot[w.same + mv]);
        else slots = a.moves[(int64_t)r * a.most + mv];
        if ((uint32_t)slots.x >= (uint32_t)m.n_slots || (uint32_t)slots.y >= (uint32_t)m.n_slots) slots = make_int2(0, -1);
        // Y layers from l on, E rows from j on; waves stay whole (verdict)
        auto move = [&](auto layers, auto rows, int l, int j) {
            constexpr int Y = decltype(layers)::value, E = decltype(rows)::value;
            for (int i0 = tid - lane; i0 < 2 * per; i0 += kWalkThreads) {
                const int i = min(i0 + lane, 2 * per - 1), x = i < per ? i : i - per, head = x >> shift, f = 8 * (x & (pieces - 1));
                auto where = [&](int y, int slot) {
                    uint16_t *const k = m.k[l + y], *const v = m.v[l + y];
                    const int row = slot & ((1 << m.page_shift) - 1);
                    return reinterpret_cast<u32x4*>((i < per ? k : v) + (slot >> m.page_shift) * m.page_stride +
                                                    (((int64_t)head << m.page_shift) + row) * m.Dh + f);
                };
                u32x4 v[Y * E];
                int to[E];
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int at = min(j + e, count64 - 1), from = __builtin_amdgcn_readlane(slots.x, at);
                    to[e] = j + e < count64 ? __builtin_amdgcn_readlane(slots.y, at) : -1;
#pragma unroll
                    for (int y = 0; y < Y; y++) v[e * Y + y] = *where(y, from);
                }
                if (status < 0) verdict();
                if (status != JH_PLAN_OK) return;
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int y = 0; y < Y; y++)
                        if (to[e] >= 0 && i0 + lane < 2 * per) *where(y, to[e]) = v[e * Y + y];
            }
        };
        using One = std::integral_constant<int, 1>;
        using Two = std::integral_constant<int, 2>;
        using Four = std::integral_constant<int, 4>;
        for (int l = (int)blockIdx.y * m.each; l < l1; l += 2)
            for (int j = 0; j < count64; j += 4) {
                if (l + 1 == l1) move(One{}, Four{}, l, j);
                else if (count64 - j == 1) move(Two{}, One{}, l, j);
                else move(Two{}, Four{}, l, j);
            }
    }
    if (!books) return;
    if (status < 0) verdict();
    const bool ok = status == JH_PLAN_OK;
    if (r == 0 && tid == 0) {
        *a.status = status;
        *a.count_out = ok ? count + total : count;
    }
    // (each row of path is written once: a refusal has nothing to take back)
    if constexpr (ONE)
        if (ok) write_path(a, 0, w, s);
    // rows that nobody has
    const int first = ok && R ? a.row_starts[0] : a.n_rows, last = ok && R ? a.row_starts[R] : a.n_rows;
    if (r == 0)
        for (int t = tid; t < first; t += kWalkThreads) a.path[t] = -1;
    if (r == R - 1)
        for (int t = last + tid; t < a.n_rows; t += kWalkThreads) a.path[t] = -1;
    if (R == 0) return;
    if (!ok) {
        if (tid == 0) a.kv_out[r] = a.kv_lens[r], a.accepted[r] = 0, a.next_tokens[r] = -1;
        return;
    }
    const int b = (int)(((int64_t)mine.w + (1 << a.page_shift) - 1) >> a.page_shift);
    for (int j = tid; j < mine.y; j += kWalkThreads) a.free_pages[count + before + j] = a.tables[(int64_t)r * a.max_blocks + b + j];
    if (tid == 0) {
        a.kv_out[r] = mine.w;
        if constexpr (ONE) a.accepted[0] = w.kept, a.next_tokens[0] = w.next;
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

size_t tree_commit_workspace_bytes(const TreeCommitArgs& a) {
    return ((size_t)a.n_req + 1) * sizeof(int4) + (size_t)a.n_req * std::min(a.tree_rows, a.n_rows) * sizeof(int2);
}

Status launch_tree_commit(TreeCommitArgs a, const TreeMoveArgs& move, void* const* k_pages, void* const* v_pages, int64_t layers,
                          void* workspace, int num_cus, hipStream_t st) {
    a.heads = static_cast<int4*>(workspace);
    a.moves = reinterpret_cast<int2*>(a.heads + a.n_req + 1);
    a.most = std::min(a.tree_rows, a.n_rows);
    // (in place, a block that begins late would find the length that another has written)
    auto apart = [](const void* x, const void* y) {
        const ptrdiff_t d = static_cast<const char*>(x) - static_cast<const char*>(y);
        return d >= (ptrdiff_t)sizeof(int32_t) || d <= -(ptrdiff_t)sizeof(int32_t);
    };
    const bool one = a.n_req == 1 && apart(a.kv_out, a.kv_lens) && apart(a.count_out, a.free_count);
    if (a.n_req && !one) hipLaunchKernelGGL(tree_walk_kernel, dim3((unsigned)a.n_req), dim3(kWalkThreads), 0, st, a);
    for (int64_t i = 0; i == 0 || i < layers; i += kMoveLayers) {
        TreeMoveArgs m = move;
        m.first = i == 0;
        m.layers = (int)std::min<int64_t>(kMoveLayers, layers - i);
        for (int j = 0; j < m.layers; j++)
            m.k[j] = static_cast<uint16_t*>(k_pages[i + j]), m.v[j] = static_cast<uint16_t*>(v_pages[i + j]);
        // about eight blocks to a CU: with fewer requests fewer layers to a block
        const int parts = std::max(1, std::min(m.layers, 8 * num_cus / std::max(1, a.n_req)));
        m.each = std::max(1, (m.layers + parts - 1) / parts);
        const unsigned y = (unsigned)std::max(1, (m.layers + m.each - 1) / m.each);
        hipLaunchKernelGGL(one ? tree_commit_kernel<true> : tree_commit_kernel<false>, dim3((unsigned)std::max(1, a.n_req), y),
                           dim3(kWalkThreads), 0, st, a, m);
    }
    return Status::ok();
}

}  // namespace jh
