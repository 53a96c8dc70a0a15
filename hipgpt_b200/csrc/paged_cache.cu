// Rows of keys and values into the pages of a cache, in its format, and back.
//
// A row is D values of one token and head.  8-bit formats hold it as codes and one fp32 scale:
//   e4m3  scale 2^k, the smallest with max|x| <= 448 * 2^k: x / scale is exact, and the code its rounding to four significant bits (to nearest even)
//   int8  scale max|x| / 127 (rounded to fp32); the code is the whole number nearest to x / scale, ties to even, of the exact quotient: the rounded product
//         with 1 / scale may be one off beside a border, and the remainder x - code * scale, which one multiply-add gives exactly, says so
//
// Bound: HBM for prompts; the launch for single tokens.  A row is read 16 bytes a thread by as many neighbouring threads as it needs (a power of two of them), the
// largest magnitude goes round by shuffles, each thread has its part of K and of V on its way at once.
#include "paged.cuh"

namespace hipgpt {
namespace {

constexpr int kThreads = 256;

struct MoveArgs {
    PagedView c;
    const void *k, *v;                   // rows of tokens (written for reading the cache)
    long long k_stride, v_stride;
    int lanes, log_lanes, vec;           // threads a row
};

// (token, head) of this thread's row, and where it lies in the cache: row < 0: nowhere; token < 0: no such row, or no sequence's
struct Place { long long token; int head; long long row; };

// The sequence of the block's first token is found by all threads together; a thread goes on from there.
__device__ __forceinline__ Place place_of(const MoveArgs &a)
{
    const long long rows = (long long)a.c.T * a.c.heads;
    const long long first = (long long)blockIdx.x << (8 - a.log_lanes);
    const int t0 = (int)(first / a.c.heads);
    int below = 0;                       // sequences that end at or before t0
    for (int b0 = 0; b0 < a.c.B; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        const int some = __syncthreads_count(b < a.c.B && __ldg(a.c.offsets + b + 1) <= t0);
        below += some;
        if (some < min(kThreads, a.c.B - b0)) break;
    }
    const long long r = first + (threadIdx.x >> a.log_lanes);
    if (r >= rows) return {-1, 0, -1};
    const int t = (int)(r / a.c.heads), head = (int)(r - (long long)t * a.c.heads);
    int b = below;
    while (b < a.c.B && __ldg(a.c.offsets + b + 1) <= t) ++b;
    if (b >= a.c.B) return {-1, 0, -1};
    const Sequence s = sequence_of(a.c, b);
    if (t < s.first || t >= s.first + s.n) return {-1, 0, -1};
    const int p = s.len - s.n + (t - s.first);
    return {t, head, p < 0 ? -1 : row_of(a.c, b, head, p)};
}

__device__ __forceinline__ float row_max(float m, int lanes)
{
    for (int o = 1; o < lanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// The scale of a row, and what its values are multiplied by in e4m3 (exact) or int8 (a first guess)
template <int FMT>
__device__ __forceinline__ float scale_of(float amax, float &inv)
{
    if constexpr (FMT == HIPGPT_CACHE_E4M3) {
        // amax = f * 2^e with 1 <= f < 2: 448 = 1.75 * 2^8
        const uint32_t u = __float_as_uint(amax);
        const int e = (int)(u >> 23) - 127, up = (u & 0x7FFFFFu) > 0x600000u;
        const int k = max(e - 8 + up, -126);
        inv = __uint_as_float((uint32_t)(127 - k) << 23);               // k <= 120
        return __uint_as_float((uint32_t)(127 + k) << 23);
    } else {
        const float s = fmaxf(__fdiv_rn(amax, 127.0f), 0x1p-126f);
        inv = __frcp_rn(s);
        return s;
    }
}
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ int int8_code(float x, float s, float inv)
{
    float q = rintf(x * inv);
    const float r = fmaf(-q, s, x), half = 0.5f * s;                    // exact: both are whole multiples of half a step of s, and |r| < s
    const bool odd = ((int)q) & 1;
    if (r > half || (r == half && odd)) q += 1.0f;
    else if (r < -half || (r == -half && odd)) q -= 1.0f;
    return (int)q;
}

template <typename T, int FMT, int W>
__global__ void __launch_bounds__(kThreads)
cache_write_kernel(const MoveArgs a)
{
    dependency_wait();
    dependents_may_start();
    const Place at = place_of(a);
    const int lane = threadIdx.x & (a.lanes - 1), D = a.c.D;
    const bool there = at.token >= 0 && at.row >= 0;
    // every thread of the warp takes part in the shuffles: those without a row have zeros
    if constexpr (W > 1) {
        const int d = lane * W;
        const bool mine = there && d < D;
        float x[2][W];
#pragma unroll
        for (int i = 0; i < W; ++i) x[0][i] = x[1][i] = 0.0f;
        if (mine) {
            load_values<T, W>(static_cast<const T *>(a.k) + at.token * a.k_stride + at.head * D + d, x[0]);
            load_values<T, W>(static_cast<const T *>(a.v) + at.token * a.v_stride + at.head * D + d, x[1]);
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint8_t *base = const_cast<uint8_t *>(w ? a.c.v : a.c.k);
            if constexpr (FMT == HIPGPT_CACHE_PLAIN) {
                if (mine) store_values<T, W>(reinterpret_cast<T *>(base) + at.row * D + d, x[w]);
            } else {
                float m = 0.0f;
                bool fine = true;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    m = fmaxf(m, fabsf(x[w][i]));
                    fine = fine && fabsf(x[w][i]) <= 3.402823466e38f;
                }
                m = row_max(fine ? m : INFINITY, a.lanes);
                float inv, s = scale_of<FMT>(m, inv);
                const bool whole = m <= 3.402823466e38f;
                uint32_t code[W / 4];
#pragma unroll
                for (int i = 0; i < W / 4; ++i) {
                    const float *y = x[w] + 4 * i;
                    if constexpr (FMT == HIPGPT_CACHE_E4M3) code[i] = e4m3_pair(y[0] * inv, y[1] * inv) | e4m3_pair(y[2] * inv, y[3] * inv) << 16;
                    else code[i] = (int8_code(y[0], s, inv) & 255) | (int8_code(y[1], s, inv) & 255) << 8 | (int8_code(y[2], s, inv) & 255) << 16 | (uint32_t)int8_code(y[3], s, inv) << 24;
                    if (!whole) code[i] = 0u;
                }
                if (mine) {
                    uint8_t *dst = base + at.row * D + d;
                    if constexpr (W == 8) *reinterpret_cast<uint2 *>(dst) = make_uint2(code[0], code[1]);
                    else *reinterpret_cast<uint32_t *>(dst) = code[0];
                    if (lane == 0) const_cast<float *>(w ? a.c.vs : a.c.ks)[at.row] = whole ? s : __uint_as_float(0x7FFFFFFFu);
                }
            }
        }
    } else {
        // rows that do not start on 16 bytes: value by value, twice
        for (int w = 0; w < 2; ++w) {
            const T *src = static_cast<const T *>(w ? a.v : a.k) + at.token * (w ? a.v_stride : a.k_stride) + at.head * D;
            uint8_t *base = const_cast<uint8_t *>(w ? a.c.v : a.c.k);
            if constexpr (FMT == HIPGPT_CACHE_PLAIN) {
                if (there) for (int d = lane; d < D; d += a.lanes) reinterpret_cast<T *>(base)[at.row * D + d] = src[d];
            } else {
                float m = 0.0f;
                if (there) for (int d = lane; d < D; d += a.lanes) {
                    const float x = fabsf(to_float(src[d]));
                    m = x <= 3.402823466e38f ? fmaxf(m, x) : INFINITY;
                }
                m = row_max(m, a.lanes);
                float inv, s = scale_of<FMT>(m, inv);
                const bool whole = m <= 3.402823466e38f;
                if (there) {
                    for (int d = lane; d < D; d += a.lanes) {
                        const float x = to_float(src[d]);
                        base[at.row * D + d] = !whole ? 0 : FMT == HIPGPT_CACHE_E4M3 ? (uint8_t)e4m3_pair(x * inv, 0.0f) : (uint8_t)int8_code(x, s, inv);
                    }
                    if (lane == 0) const_cast<float *>(w ? a.c.vs : a.c.ks)[at.row] = whole ? s : __uint_as_float(0x7FFFFFFFu);
                }
            }
        }
    }
}

template <typename T, int FMT, int W>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const MoveArgs a)
{
    dependency_wait();
    dependents_may_start();
    const Place at = place_of(a);
    if (at.token < 0) return;
    const int D = a.c.D;
    const bool there = at.row >= 0;
    constexpr int STEP = W > 1 ? W : 1;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const uint8_t *base = w ? a.c.v : a.c.k;
        T *dst = static_cast<T *>(const_cast<void *>(w ? a.v : a.k)) + at.token * (w ? a.v_stride : a.k_stride) + at.head * D;
        float s = 0.0f;
        if constexpr (FMT != HIPGPT_CACHE_PLAIN) if (there) s = __ldg((w ? a.c.vs : a.c.ks) + at.row);
        for (int d = (threadIdx.x & (a.lanes - 1)) * STEP; d < D; d += a.lanes * STEP) {
            float x[STEP];
#pragma unroll
            for (int i = 0; i < STEP; ++i) x[i] = 0.0f;
            if (there) {
                if constexpr (FMT == HIPGPT_CACHE_PLAIN) {
                    load_values<T, STEP>(reinterpret_cast<const T *>(base) + at.row * D + d, x);
                } else if constexpr (W == 1) {
                    const uint32_t two = code_pair<FMT>(base[at.row * D + d], 0u, 0, 0);
                    x[0] = __uint_as_float(two << 16) * s;
                } else {
                    uint32_t word[W / 4];
                    if constexpr (W == 8) {
                        const uint2 u = *reinterpret_cast<const uint2 *>(base + at.row * D + d);
                        word[0] = u.x; word[1] = u.y;
                    } else {
                        word[0] = *reinterpret_cast<const uint32_t *>(base + at.row * D + d);
                    }
#pragma unroll
                    for (int i = 0; i < W / 2; ++i) {
                        const uint32_t two = code_pair<FMT>(word[i / 2], word[i / 2], (i & 1) * 2, (i & 1) * 2 + 1);
                        x[2 * i] = __uint_as_float(two << 16) * s;
                        x[2 * i + 1] = __uint_as_float(two & 0xFFFF0000u) * s;
                    }
                }
            }
            store_values<T, STEP>(dst + d, x);
        }
    }
}

template <typename T, int FMT>
int launch_move(MoveArgs a, bool write, cudaStream_t st)
{
    constexpr int W = kPer16<T>;
    const bool vec = all_aligned16({a.k, a.v}) && a.k_stride % W == 0 && a.v_stride % W == 0;
    // D / W threads of 16 bytes, rounded up to a power of two; without them as many as a warp
    a.log_lanes = 0;
    while (a.log_lanes < 5 && (vec ? W : 4) << a.log_lanes < a.c.D) ++a.log_lanes;
    a.lanes = 1 << a.log_lanes;
    const long long rows = (long long)a.c.T * a.c.heads, per = kThreads >> a.log_lanes, blocks = (rows + per - 1) / per;
    if (blocks > 2147483647LL) return fail(HIPGPT_ERR_BAD_ARG, "%d tokens of %d heads are beyond one call", a.c.T, a.c.heads);
    const auto kern = write ? (vec ? cache_write_kernel<T, FMT, W> : cache_write_kernel<T, FMT, 1>) : (vec ? cache_read_kernel<T, FMT, W> : cache_read_kernel<T, FMT, 1>);
    const cudaError_t e = launch_overlapped(kern, dim3((unsigned)blocks), dim3(kThreads), 0, st, a);
    const char *what = write ? "cache_write_kernel" : "cache_read_kernel";
    return e == cudaSuccess ? check_launch(what) : fail(HIPGPT_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
template <typename T>
int launch_move_of(int format, const MoveArgs &a, bool write, cudaStream_t st)
{
    return format == HIPGPT_CACHE_PLAIN ? launch_move<T, HIPGPT_CACHE_PLAIN>(a, write, st)
         : format == HIPGPT_CACHE_E4M3  ? launch_move<T, HIPGPT_CACHE_E4M3>(a, write, st) : launch_move<T, HIPGPT_CACHE_INT8>(a, write, st);
}

int move_rows(const hipgpt_paged_cache *cache, const hipgpt_paged_batch *batch, const void *k, long long k_stride, const void *v, long long v_stride, bool write, void *stream)
{
    MoveArgs a = {};
    const int rc = check_paged(cache, batch, &a.c);
    if (rc != HIPGPT_OK) return rc > 0 ? HIPGPT_OK : rc;
    if (!k || !v) return fail(HIPGPT_ERR_NULL, "k and v must not be NULL");
    const long long width = (long long)cache->heads * cache->head_dim;
    if (check_stride("k", k_stride, width) != HIPGPT_OK || check_stride("v", v_stride, width) != HIPGPT_OK) return HIPGPT_ERR_BAD_ARG;
    const size_t es = cache->type == HIPGPT_TYPE_F32 ? 4 : 2;
    const Rows rk{k, (size_t)k_stride * es, (size_t)width * es, batch->tokens}, rv{v, (size_t)v_stride * es, (size_t)width * es, batch->tokens};
    if (write) {
        // the cache's four arrays are written
        const size_t rows = cache_rows(cache), bytes = rows * cache->head_dim * cache_element_bytes(cache), scales = cache->format == HIPGPT_CACHE_PLAIN ? 0 : rows * 4;
        const int over = refuse_overlaps(4, {{cache->k, bytes}, {cache->v, bytes}, {cache->k_scale, scales}, {cache->v_scale, scales}, {k, extent_of(rk)}, {v, extent_of(rv)},
                                             {batch->offsets, 4 * ((size_t)batch->sequences + 1)}, {batch->lengths, 4 * (size_t)batch->sequences},
                                             {batch->page_table, 4 * (size_t)batch->sequences * batch->most_pages}});
        if (over != HIPGPT_OK) return over;
    } else {
        int over = refuse_rows_over(rk, {rv}, cache, batch);
        if (over == HIPGPT_OK) over = refuse_rows_over(rv, {}, cache, batch);
        if (over != HIPGPT_OK) return over;
    }
    a.k = k; a.v = v;
    a.k_stride = k_stride; a.v_stride = v_stride;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return cache->type == HIPGPT_TYPE_F32 ? launch_move_of<float>(cache->format, a, write, st) : launch_move_of<__nv_bfloat16>(cache->format, a, write, st);
}

}  // namespace
}  // namespace hipgpt

using namespace hipgpt;

extern "C" int hipgpt_cache_write(const hipgpt_paged_cache *cache, const hipgpt_paged_batch *batch, const void *d_k, long long k_stride, const void *d_v, long long v_stride, void *stream)
{
    return move_rows(cache, batch, d_k, k_stride, d_v, v_stride, true, stream);
}

extern "C" int hipgpt_cache_read(const hipgpt_paged_cache *cache, const hipgpt_paged_batch *batch, void *d_k, long long k_stride, void *d_v, long long v_stride, void *stream)
{
    return move_rows(cache, batch, d_k, k_stride, d_v, v_stride, false, stream);
}
