// Embedding lookup with a scale, for fp32 and bf16 tables, and its gradient (HipGPT's launch_embedding_lookup and
// embedding_backward_kernel, src/hip_kernels.cpp:537-599 and :1064-1088; the reference adds its gradients with atomics, in any order).
//
//   out[t]      = scale tok[id_t] + pos[t mod S]                       an id outside [0, V) gives a row of zeros
//   grad_tok[v] = scale * sum of g[t] over the t with id_t = v         (+ what it held, when accumulating)
//   grad_pos[s] = sum of g[b S + s] over the b whose id is inside      (likewise)
//
// Both are bound by HBM: rows read once, rows written once.
//
// The gradient sums every row of the table in a fixed order, without atomics on values: the tokens are sorted by id first.
//   sort_ids_kernel   one cluster of sixteen blocks sorts (id, t) by id, stable (so equal ids keep ascending t): two passes of
//                     counting sort for vocabularies up to 2^20, three beyond; then writes where the entries of each row begin.
//                     Within a pass a block counts its part's digits, the cluster's counts become offsets through
//                     distributed shared memory, and every warp ranks 32 keys at a time among themselves (match).
//   embed_sum_kernel  a group of up to 32 lanes takes 16 bytes a lane of one row of the table: adds its entries and stores the row, zeros
//                     where there are none.  Words are not spread evenly (one id may take a tenth of the tokens, padding half of them), so a
//                     row of more than C entries is summed in pieces of C by many groups; the group that finishes a row's last piece
//                     adds the pieces, in ascending order whichever group it is.  The positions' table is summed in the same way over the batch.
#include "elem_types.cuh"
#include "stream_workspace.hpp"

namespace hipgpt {
namespace {

// ---- lookup -----------------------------------------------------------------------------------------------------------

// One warp per row, 16 bytes a lane (W = 1: value by value).
template <typename T, int W, bool POS>
__global__ void __launch_bounds__(256)
embedding_scaled_kernel(const int *__restrict__ ids, const T *__restrict__ tok, const T *__restrict__ pos, T *__restrict__ out, float scale, long long n, int S, int V, int E)
{
    dependency_wait();
    dependents_may_start();
    const int lane = threadIdx.x & 31;
    const long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (t >= n) return;
    const int id = ids[t];
    const bool ok = id >= 0 && id < V;
    const T *src = tok + (size_t)(ok ? id : 0) * E, *prow = POS ? pos + (size_t)(t % S) * E : nullptr;
    T *dst = out + (size_t)t * E;
#pragma unroll 4
    for (int e = lane * W; e < E; e += 32 * W) {
        float x[W], p[W];
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] = p[j] = 0.0f;
        if (ok) {
            load_values<T, W>(src + e, x);
            if constexpr (POS) load_values<T, W>(prow + e, p);
#pragma unroll
            for (int j = 0; j < W; ++j) x[j] = POS ? __fadd_rn(__fmul_rn(scale, x[j]), p[j]) : __fmul_rn(scale, x[j]);
        }
        store_values<T, W>(dst + e, x);
    }
}

template <typename T>
int launch_embedding_scaled(const int *ids, const void *tok, const void *pos, void *out, float scale, long long n, int S, int V, int E, cudaStream_t st)
{
    constexpr int W = kPer16<T>;
    const bool vec = E % W == 0 && all_aligned16({tok, pos, out});
    const auto kern = pos ? (vec ? embedding_scaled_kernel<T, W, true> : embedding_scaled_kernel<T, 1, true>)
                          : (vec ? embedding_scaled_kernel<T, W, false> : embedding_scaled_kernel<T, 1, false>);
    const cudaError_t e = launch_overlapped(kern, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, st, ids, static_cast<const T *>(tok), static_cast<const T *>(pos), static_cast<T *>(out),
                                            scale, n, S, V, E);
    return e == cudaSuccess ? check_launch("embedding_scaled_kernel") : fail(HIPGPT_ERR_CUDA, "embedding_scaled_kernel: %s", cudaGetErrorString(e));
}

// ---- the tokens in the order of their ids -----------------------------------------------------------------------------

constexpr int kSortBlocks = 16, kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kKeysPerLane = 4, kWarpKeys = 32 * kKeysPerLane, kTileKeys = kSortWarps * kWarpKeys;
constexpr int kMostBits = 10, kMostBins = 1 << kMostBits;

struct SortShared {
    int hist[kMostBins];                    // digits of this block's part; read by the other blocks
    int base[kMostBins];                    // where this block's next key of each digit goes
    unsigned short warp_count[kSortWarps][kMostBins];
    int warp_sum[kSortWarps];
};

__device__ __forceinline__ int read_peer_int(const int *p, int rank)
{
    int v;
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(peer_addr(smem_u32(p), rank)) : "memory");
    return v;
}

// ids [n] -> (id, t) sorted in `sorted` (ids outside [0, V) as V, last), row_start[v] = first entry of row v (v <= V; row_start[V] = entries inside), and
// counters[0 .. ncounters) = 0.  `other`: a second buffer of n entries.  npass passes of `bits` bits; the last one ends in `sorted`.
__global__ void __launch_bounds__(kSortThreads)
sort_ids_kernel(const int *__restrict__ ids, int n, int V, int bits, int npass, int2 *sorted, int2 *other, int *row_start, int *counters, int ncounters)
{
    extern __shared__ __align__(16) uint8_t sort_smem[];
    SortShared &s = *reinterpret_cast<SortShared *>(sort_smem);
    const int rank = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int bins = 1 << bits;
    dependency_wait();
    dependents_may_start();
    for (int i = rank * kSortThreads + tid; i < ncounters; i += kSortBlocks * kSortThreads) counters[i] = 0;
    const int per = ((n + kSortBlocks - 1) / kSortBlocks + 31) / 32 * 32;
    const int from = min((long long)rank * per, (long long)n), to = min((long long)from + per, (long long)n);
    const int2 *src = nullptr;
    for (int pass = 0; pass < npass; ++pass) {
        const int shift = pass * bits;
        int2 *dst = (npass - pass) & 1 ? sorted : other;
        for (int d = tid; d < bins; d += kSortThreads) s.hist[d] = 0;
        __syncthreads();
        auto entry = [&](int i) {
            if (pass) return __ldcg(src + i);
            const int id = ids[i];
            return make_int2(id >= 0 && id < V ? id : V, i);
        };
        for (int i = from + tid; i < to; i += kSortThreads) atomicAdd(&s.hist[entry(i).x >> shift & (bins - 1)], 1);
        cluster_sync();
        // digit d = tid: keys of smaller digits anywhere, and of this digit in the blocks before
        int total = 0, before = 0;
        if (tid < bins)
#pragma unroll
            for (int r = 0; r < kSortBlocks; ++r) {
                const int h = read_peer_int(&s.hist[tid], r);
                total += h;
                before += r < rank ? h : 0;
            }
        int incl = total;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) s.warp_sum[warp] = incl;
        __syncthreads();
        int prev = 0;
        for (int w = 0; w < warp; ++w) prev += s.warp_sum[w];
        if (tid < bins) s.base[tid] = prev + incl - total + before;
        for (int t0 = from; t0 < to; t0 += kTileKeys) {
            __syncthreads();
            for (int i = tid; i < kSortWarps * bins; i += kSortThreads) s.warp_count[i >> bits][i & (bins - 1)] = 0;
            __syncthreads();
            int2 e[kKeysPerLane];
            int place[kKeysPerLane];
#pragma unroll
            for (int k = 0; k < kKeysPerLane; ++k) {
                const int i = t0 + warp * kWarpKeys + k * 32 + lane;
                e[k] = i < to ? entry(i) : make_int2(-1, 0);
            }
#pragma unroll
            for (int k = 0; k < kKeysPerLane; ++k) {
                const int d = e[k].x < 0 ? -1 : e[k].x >> shift & (bins - 1);
                const unsigned same = __match_any_sync(0xffffffffu, d);
                const int mine = __popc(same & ((1u << lane) - 1));
                const int seen = d >= 0 ? s.warp_count[warp][d] : 0;
                __syncwarp();
                place[k] = seen + mine;
                if (d >= 0 && mine == 0) s.warp_count[warp][d] = (unsigned short)(seen + __popc(same));
                __syncwarp();
            }
            __syncthreads();
            // counts of the warps -> offsets among them; the next tile begins behind this one
            int all = 0;
            if (tid < bins) {
                for (int w = 0; w < kSortWarps; ++w) {
                    const int c = s.warp_count[w][tid];
                    s.warp_count[w][tid] = (unsigned short)all;
                    all += c;
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kKeysPerLane; ++k)
                if (e[k].x >= 0) {
                    const int d = e[k].x >> shift & (bins - 1);
                    __stcg(dst + s.base[d] + s.warp_count[warp][d] + place[k], e[k]);
                }
            __syncthreads();
            if (tid < bins) s.base[tid] += all;
        }
        __threadfence();
        cluster_sync();                      // the pass's entries are all there, and nobody reads this block's counts any more
        src = dst;
    }
    // rows between one entry's id and the next begin at the next; each warp fills the gaps of 32 entries together
    for (int i0 = from + warp * 32; i0 < to; i0 += kSortThreads) {
        const int i = i0 + lane;
        const int key = i < n ? __ldcg(&src[i].x) : V, prev = i == 0 ? -1 : i <= n ? __ldcg(&src[i - 1].x) : V;
        const bool live = i < to;
        unsigned gaps = __ballot_sync(0xffffffffu, live && key > prev);
        while (gaps) {
            const int l = __ffs(gaps) - 1;
            gaps &= gaps - 1;
            const int a = __shfl_sync(0xffffffffu, prev, l) + 1, b = __shfl_sync(0xffffffffu, key, l), at = i0 + l;
            for (int v = a + lane; v <= b; v += 32) row_start[v] = at;
        }
    }
    if (rank == 0) {                          // rows behind the last entry
        const int last = __ldcg(&src[n - 1].x);
        for (int v = last + 1 + tid; v <= V; v += kSortThreads) row_start[v] = n;
    }
}

// ---- sums of rows -----------------------------------------------------------------------------------------------------

// Where the work of embed_sum_kernel lies.  Tasks of one group (2^lanes_log lanes, W values each: `slices` of them cover a row) in this order: pieces of
// long rows, pieces of the batch of the positions' rows, rows.
struct SumPlan {
    int n, V, E, B, S;
    int slices, lanes_log;
    int piece, pieces;                        // entries of a piece of a long row; pieces of all entries
    int pos_piece, pos_pieces;                // batches of a piece of a position's row, and how many; 0: no positions' table
    long long pos_first, row_first, tasks;
};

template <typename G, int W>
__device__ __forceinline__ void put_row(G *p, float (&v)[W], float scale, bool accumulate)
{
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = __fmul_rn(v[j], scale);
    if (accumulate) {
        float old[W];
        load_values<G, W>(p, old);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = __fadd_rn(old[j], v[j]);
    }
    store_values<G, W>(p, v);
}

// The lanes of a group that has stored its piece's sum: whether it is the last of `pieces` to do so (the others' sums are then visible)
__device__ __forceinline__ bool last_piece(int *counter, int pieces, unsigned mask, int leader)
{
    __threadfence();
    __syncwarp(mask);
    int seen = 0;
    if ((int)(threadIdx.x & 31) == leader) seen = atomicAdd(counter, 1);
    seen = __shfl_sync(mask, seen, leader);
    __threadfence();
    return seen == pieces - 1;
}

template <int W>
__device__ __forceinline__ void add(float (&a)[W], const float (&b)[W])
{
#pragma unroll
    for (int j = 0; j < W; ++j) a[j] = __fadd_rn(a[j], b[j]);
}

template <typename T, typename G, int W>
__global__ void __launch_bounds__(256)
embed_sum_kernel(const T *__restrict__ g, const int *__restrict__ ids, const int2 *__restrict__ sorted, const int *__restrict__ row_start, float *part, float *pos_part, int *counters,
                 G *grad_tok, G *grad_pos, float scale, int accumulate, SumPlan p)
{
    dependency_wait();
    dependents_may_start();
    const int lanes = 1 << p.lanes_log, lane = threadIdx.x & 31, sub = lane & (lanes - 1), leader = lane - sub;
    const unsigned mask = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1) << leader;
    const long long task = ((long long)blockIdx.x * 256 + threadIdx.x) >> p.lanes_log;
    if (task >= p.tasks) return;
    constexpr int kAhead = W == 1 ? 8 : 4;
    float acc[W];
#pragma unroll
    for (int j = 0; j < W; ++j) acc[j] = 0.0f;
    // rows a .. b of the sorted entries, in order
    auto sum_entries = [&](int a, int b, int e) {
        int i = a;
        for (; i + kAhead <= b; i += kAhead) {
            float x[kAhead][W];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) load_values<T, W>(g + (size_t)__ldg(&sorted[i + k].y) * p.E + e, x[k]);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) add(acc, x[k]);
        }
        for (; i < b; ++i) {
            float x[W];
            load_values<T, W>(g + (size_t)__ldg(&sorted[i].y) * p.E + e, x);
            add(acc, x);
        }
    };
    auto sum_parts = [&](const float *first, size_t stride, int count) {
#pragma unroll
        for (int j = 0; j < W; ++j) acc[j] = 0.0f;
        int i = 0;
        for (; i + 8 <= count; i += 8) {
            float x[8][W];
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int j = 0; j < W; ++j) x[k][j] = __ldcg(first + (i + k) * stride + j);
#pragma unroll
            for (int k = 0; k < 8; ++k) add(acc, x[k]);
        }
        for (; i < count; ++i) {
            float x[W];
#pragma unroll
            for (int j = 0; j < W; ++j) x[j] = __ldcg(first + i * stride + j);
            add(acc, x);
        }
    };
    if (task >= p.row_first) {
        const long long r = task - p.row_first;
        const int v = (int)(r / p.slices), e = ((int)(r % p.slices) * lanes + sub) * W;
        if (e >= p.E) return;
        const int a = __ldg(row_start + v), b = __ldg(row_start + v + 1);
        if (b - a > p.piece || (accumulate && a == b)) return;      // summed in pieces; nothing to add
        sum_entries(a, b, e);
        put_row<G, W>(grad_tok + (size_t)v * p.E + e, acc, scale, accumulate != 0);
        return;
    }
    if (task < p.pos_first) {
        // a piece of the sorted entries: at most one long row ends or passes in it, and at most one begins
        const int c = (int)(task / p.slices), sl = (int)(task % p.slices), e0 = (sl * lanes + sub) * W, e = e0 < p.E ? e0 : 0;      // (a lane past the row sums its first values for nothing: its group meets in the counting)
        const int c0 = c * p.piece, c1 = min(p.n, c0 + p.piece);
        int i = c0;
        while (i < c1) {
            const int v = __ldg(&sorted[i].x);
            if (v >= p.V) return;
            const int a = __ldg(row_start + v), b = __ldg(row_start + v + 1);
            if (b - a > p.piece) {
                const int first = a / p.piece, count = (b - 1) / p.piece - first + 1;
#pragma unroll
                for (int j = 0; j < W; ++j) acc[j] = 0.0f;
                sum_entries(max(a, c0), min(b, c1), e);
                // a piece's sum of the row that was there before it, and of the one that begins in it
                if (e0 < p.E)
#pragma unroll
                    for (int j = 0; j < W; ++j) __stcg(part + (size_t)(2 * c + (c == first)) * p.E + e + j, acc[j]);
                if (last_piece(counters + first * p.slices + sl, count, mask, leader) && e0 < p.E) {
                    sum_parts(part + (size_t)(2 * first + 1) * p.E + e, 0, 1);
                    float head[W];
#pragma unroll
                    for (int j = 0; j < W; ++j) head[j] = acc[j];
                    sum_parts(part + (size_t)(2 * (first + 1)) * p.E + e, 2 * (size_t)p.E, count - 1);
                    add(head, acc);
                    put_row<G, W>(grad_tok + (size_t)v * p.E + e, head, scale, accumulate != 0);
                }
            }
            i = b;
        }
        return;
    }
    {
        const long long r = task - p.pos_first;
        const int sl = (int)(r % p.slices), e0 = (sl * lanes + sub) * W, e = e0 < p.E ? e0 : 0;
        const int s = (int)(r / p.slices % p.S), c = (int)(r / p.slices / p.S);
        const int b0 = c * p.pos_piece, b1 = min(p.B, b0 + p.pos_piece);
        int b = b0;
        for (; b + kAhead <= b1; b += kAhead) {
            float x[kAhead][W];
            bool ok[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const size_t t = (size_t)(b + k) * p.S + s;
                const int id = __ldg(ids + t);
                ok[k] = id >= 0 && id < p.V;
                load_values<T, W>(g + t * p.E + e, x[k]);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) if (ok[k]) add(acc, x[k]);
        }
        for (; b < b1; ++b) {
            const size_t t = (size_t)b * p.S + s;
            const int id = __ldg(ids + t);
            float x[W];
            load_values<T, W>(g + t * p.E + e, x);
            if (id >= 0 && id < p.V) add(acc, x);
        }
        G *dst = grad_pos + (size_t)s * p.E + e;
        if (p.pos_pieces == 1) {
            if (e0 < p.E) put_row<G, W>(dst, acc, 1.0f, accumulate != 0);
            return;
        }
        const size_t row = (size_t)s * p.E + e, stride = (size_t)p.S * p.E;
        if (e0 < p.E)
#pragma unroll
            for (int j = 0; j < W; ++j) __stcg(pos_part + c * stride + row + j, acc[j]);
        if (last_piece(counters + p.pieces * p.slices + s * p.slices + sl, p.pos_pieces, mask, leader) && e0 < p.E) {
            sum_parts(pos_part + row, stride, p.pos_pieces);
            put_row<G, W>(dst, acc, 1.0f, accumulate != 0);
        }
    }
}

StreamWorkspace g_embed_ws;

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
size_t padded(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

template <typename T, typename G>
int launch_embedding_backward(const void *grad_out, const int *ids, void *grad_tok, void *grad_pos, float scale, int accumulate, int B, int S, int V, int E, cudaStream_t st)
{
    const int n = B * S;
    // what a piece holds: long enough that few rows come in pieces, short enough that the last of a row's pieces is no long sum over the others
    SumPlan p = {};
    p.n = n; p.V = V; p.E = E; p.B = B; p.S = S;
    const bool vec = E % kPer16<T> == 0 && all_aligned16({grad_out, grad_tok, grad_pos});
    const int W = vec ? kPer16<T> : 1, words = ceil_div(E, W);
    while ((1 << p.lanes_log) < words && p.lanes_log < 5) ++p.lanes_log;
    p.slices = ceil_div(words, 1 << p.lanes_log);
    p.piece = n > 65536 ? (n / 1024 + 31) / 32 * 32 : 64;
    p.pieces = ceil_div(n, p.piece);
    p.pos_piece = B > 4096 ? B / 64 : 64;
    p.pos_pieces = grad_pos ? ceil_div(B, p.pos_piece) : 0;
    p.pos_first = grad_tok ? (long long)p.pieces * p.slices : 0;
    p.row_first = p.pos_first + (long long)p.pos_pieces * S * p.slices;
    p.tasks = p.row_first + (grad_tok ? (long long)V * p.slices : 0);
    const long long blocks = ((p.tasks << p.lanes_log) + 255) / 256;
    const long long ncounters = (long long)p.pieces * p.slices + (p.pos_pieces > 1 ? (long long)S * p.slices : 0);
    if (blocks > 2147483647LL || ncounters > 2147483647LL) return fail(HIPGPT_ERR_UNSUPPORTED, "a table of %d rows of %d values is beyond one call", V, E);

    const size_t entry_bytes = padded((size_t)n * sizeof(int2)), start_bytes = padded(((size_t)V + 1) * sizeof(int)), counter_bytes = padded((size_t)ncounters * sizeof(int));
    const size_t part_bytes = padded((size_t)2 * p.pieces * E * sizeof(float)), pos_bytes = p.pos_pieces > 1 ? padded((size_t)p.pos_pieces * S * E * sizeof(float)) : 0;
    StreamWorkspace::Lease ws;
    int rc = g_embed_ws.enter(st, 2 * entry_bytes + start_bytes + counter_bytes + part_bytes + pos_bytes, &ws);
    if (rc != HIPGPT_OK) return rc;
    uint8_t *at = ws.get();
    auto take = [&](size_t bytes) { uint8_t *r = at; at += bytes; return r; };
    int2 *sorted = reinterpret_cast<int2 *>(take(entry_bytes)), *other = reinterpret_cast<int2 *>(take(entry_bytes));
    int *row_start = reinterpret_cast<int *>(take(start_bytes)), *counters = reinterpret_cast<int *>(take(counter_bytes));
    float *part = reinterpret_cast<float *>(take(part_bytes)), *pos_part = reinterpret_cast<float *>(take(pos_bytes));

    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    static std::atomic<unsigned long long> done{0};
    if (e == cudaSuccess) e = once_per_device(done, dev, [] {
        cudaError_t r = cudaFuncSetAttribute(sort_ids_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortShared));
        if (r == cudaSuccess) r = cudaFuncSetAttribute(sort_ids_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        return r;
    });
    int key_bits = 1;
    while (key_bits < 31 && (V >> key_bits)) ++key_bits;                   // keys 0 ... V
    const int npass = ceil_div(key_bits, kMostBits), bits = ceil_div(key_bits, npass);
    if (!grad_tok) {                                                       // no order is asked for; nothing of the long rows runs
        if (e == cudaSuccess) e = cudaMemsetAsync(counters, 0, (size_t)ncounters * sizeof(int), st);
    } else if (e == cudaSuccess) e = launch_overlapped_clusters(sort_ids_kernel, kSortBlocks, dim3(kSortBlocks), dim3(kSortThreads), sizeof(SortShared), st, ids, n, V, bits, npass, sorted, other, row_start,
                                                         counters, (int)ncounters);
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "sort_ids_kernel: %s", cudaGetErrorString(e));
    rc = check_launch("sort_ids_kernel");
    if (rc != HIPGPT_OK) return rc;
    const auto kern = vec ? embed_sum_kernel<T, G, kPer16<T>> : embed_sum_kernel<T, G, 1>;
    e = launch_overlapped(kern, dim3((unsigned)blocks), dim3(256), 0, st, static_cast<const T *>(grad_out), ids, (const int2 *)sorted, (const int *)row_start, part, pos_part, counters,
                          static_cast<G *>(grad_tok), static_cast<G *>(grad_pos), scale, accumulate, p);
    return e == cudaSuccess ? check_launch("embed_sum_kernel") : fail(HIPGPT_ERR_CUDA, "embed_sum_kernel: %s", cudaGetErrorString(e));
}

int check_embedding_sizes(int B, int S, int V, int E, int type)
{
    if (type != HIPGPT_TYPE_F32 && type != HIPGPT_TYPE_BF16) return fail(HIPGPT_ERR_BAD_ARG, "unknown type %d", type);
    if (B < 0 || S < 0 || V < 0 || E < 0) return fail(HIPGPT_ERR_BAD_ARG, "negative size: B=%d S=%d V=%d E=%d", B, S, V, E);
    if ((long long)B * S > 1LL << 30) return fail(HIPGPT_ERR_UNSUPPORTED, "%lld tokens are beyond one call", (long long)B * S);
    return HIPGPT_OK;
}

}  // namespace

void embedding_release_scratch() { g_embed_ws.release(); }

}  // namespace hipgpt

using namespace hipgpt;

extern "C" {

int hipgpt_embedding_scaled(const int *d_ids, const void *d_tok, const void *d_pos, void *d_out, float scale, int B, int S, int V, int E, int type, void *stream)
{
    const int rc = check_embedding_sizes(B, S, V, E, type);
    if (rc != HIPGPT_OK) return rc;
    if (B == 0 || S == 0 || E == 0) return HIPGPT_OK;
    if (!d_ids || !d_out || (V > 0 && !d_tok)) return fail(HIPGPT_ERR_NULL, "ids, tok and out must not be NULL");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return type == HIPGPT_TYPE_F32 ? launch_embedding_scaled<float>(d_ids, d_tok, d_pos, d_out, scale, (long long)B * S, S, V, E, st)
                                   : launch_embedding_scaled<__nv_bfloat16>(d_ids, d_tok, d_pos, d_out, scale, (long long)B * S, S, V, E, st);
}

int hipgpt_embedding_backward(const void *d_grad_out, const int *d_ids, void *d_grad_tok, void *d_grad_pos, float scale, int accumulate,
                              int B, int S, int V, int E, int type, int grad_type, void *stream)
{
    const int rc = check_embedding_sizes(B, S, V, E, type);
    if (rc != HIPGPT_OK) return rc;
    if (grad_type != HIPGPT_TYPE_F32 && grad_type != HIPGPT_TYPE_BF16) return fail(HIPGPT_ERR_BAD_ARG, "unknown type %d", grad_type);
    if (type == HIPGPT_TYPE_F32 && grad_type == HIPGPT_TYPE_BF16) return fail(HIPGPT_ERR_UNSUPPORTED, "fp32 gradients are not summed into bf16 tables");
    if (E == 0 || (!d_grad_tok && !d_grad_pos)) return HIPGPT_OK;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t gs = grad_type == HIPGPT_TYPE_F32 ? 4 : 2;
    if (B == 0 || S == 0) {                              // no token: gradients of zero
        if (accumulate) return HIPGPT_OK;
        cudaError_t e = d_grad_tok && V ? cudaMemsetAsync(d_grad_tok, 0, (size_t)V * E * gs, st) : cudaSuccess;
        if (e == cudaSuccess && d_grad_pos && S) e = cudaMemsetAsync(d_grad_pos, 0, (size_t)S * E * gs, st);
        return e == cudaSuccess ? HIPGPT_OK : fail(HIPGPT_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
    }
    if (!d_grad_out || !d_ids) return fail(HIPGPT_ERR_NULL, "grad_out and ids must not be NULL");
    if (type == HIPGPT_TYPE_F32) return launch_embedding_backward<float, float>(d_grad_out, d_ids, d_grad_tok, d_grad_pos, scale, accumulate, B, S, V, E, st);
    return grad_type == HIPGPT_TYPE_F32 ? launch_embedding_backward<__nv_bfloat16, float>(d_grad_out, d_ids, d_grad_tok, d_grad_pos, scale, accumulate, B, S, V, E, st)
                                        : launch_embedding_backward<__nv_bfloat16, __nv_bfloat16>(d_grad_out, d_ids, d_grad_tok, d_grad_pos, scale, accumulate, B, S, V, E, st);
}

}  // extern "C"
