// Rows of keys and values into the pages of a cache, in its format, and back.
//
// A row is D values of one token and head.  8-bit formats hold it as codes and one fp32 scale:
//   e4m3  scale 2^k, the smallest with max|x| <= 448 * 2^k: x / scale is exact, and the code its rounding to four significant bits (to nearest even)
//   int8  scale max|x| / 127 (rounded to fp32); the code is the whole number nearest to x / scale, ties to even, of the exact quotient: the rounded product
//         with 1 / scale may be one off beside a border, and the remainder x - code * scale, which one multiply-add gives exactly, says so
//
// Bound: issue slots of the conversion to codes, then HBM, for prompts (12 of up to 4096 tokens, 8 heads of 128, bf16 to int8 and back: 92 us, 4.5 TB/s; 172 us with a look-up for each row and rounding by the
// special-function unit); the launch for single tokens (64 tokens written and read: 7.3 us).  A block takes some tokens; where each goes is looked up once for all its heads.  A row is read 16 bytes a thread by as many neighbouring
// threads as it needs (a power of two of them), the largest magnitude goes round by shuffles, and a thread has its parts of K and of V on their way at once.
#include "paged.cuh"

namespace hipgpt {
namespace {

constexpr int kThreads = 256, kMostTokens = 32;

struct MoveArgs {
    PagedView c;
    const void *k, *v;                   // rows of tokens (written for reading the cache)
    long long k_stride, v_stride;
    int lanes, log_lanes, tokens;        // threads a row; tokens a block
    uint32_t per_head;                   // 2^32 / heads, rounded up: r * per_head >> 32 is r / heads for r * heads < 2^32
};

// Where the block's tokens lie in the cache: the row of head 0 (the others 1 << shift apart), -1: nowhere, -2: no such token, or no sequence's.  The sequence of the first is found
// by all threads together; a thread for each token goes on from there.
__device__ __forceinline__ void places_of(const MoveArgs &a, int t0, long long (&places)[kMostTokens])
{
    int below = 0;                       // sequences that end at or before t0
    for (int b0 = 0; b0 < a.c.B; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        const int some = __syncthreads_count(b < a.c.B && __ldg(a.c.offsets + b + 1) <= t0);
        below += some;
        if (some < min(kThreads, a.c.B - b0)) break;
    }
    if ((int)threadIdx.x < a.tokens) {
        long long place = -2;
        if ((int)threadIdx.x < a.c.T - t0) {         // (t0 + 31 may be beyond an int)
            const int t = t0 + threadIdx.x;
            int b = below;
            while (b < a.c.B && __ldg(a.c.offsets + b + 1) <= t) ++b;
            if (b < a.c.B) {
                const Sequence s = sequence_of(a.c, b);
                if (t >= s.first && t < s.first + s.n) {
                    const int p = s.len - s.n + (t - s.first);
                    place = p < 0 ? -1 : row_of(a.c, b, 0, p);
                }
            }
        }
        places[threadIdx.x] = place;
    }
    __syncthreads();
}

// Magnitudes as their bits: of numbers in their order, infinities and NaN above all of them
__device__ __forceinline__ uint32_t row_max(uint32_t m, int lanes)
{
    for (int o = 1; o < lanes; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
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
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));        // (2^-23 of it: a guess)
        return s;
    }
}
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Four codes of a word.  x * inv + 1.5 * 2^23 rounds to the nearest whole number in the low bits; x * inv is off by 127 * 2^-23 of a code at most, so only where a remainder
// comes within 4 * 10^-5 of half a scale, which is seldom, the four are looked at again.
__device__ __forceinline__ int int8_code(float x, float s, float inv)
{
    float q = rintf(x * inv);
    const float r = fmaf(-q, s, x), half = 0.5f * s;                    // exact: both are whole multiples of half a step of s, and |r| < s
    const bool odd = ((int)q) & 1;
    if (r > half || (r == half && odd)) q += 1.0f;
    else if (r < -half || (r == -half && odd)) q -= 1.0f;
    return (int)q;
}
__device__ __forceinline__ uint32_t int8_word(const float *x, float s, float inv)
{
    constexpr float kMagic = 12582912.0f;
    float t[4], far = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        t[e] = fmaf(x[e], inv, kMagic);
        far = fmaxf(far, fabsf(fmaf(kMagic - t[e], s, x[e])));
    }
    uint32_t w = __byte_perm(__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040), __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
    if (far > 0.49996f * s) w = (int8_code(x[0], s, inv) & 255) | (int8_code(x[1], s, inv) & 255) << 8 | (int8_code(x[2], s, inv) & 255) << 16 | (uint32_t)int8_code(x[3], s, inv) << 24;
    return w;
}

// A thread takes two chunks of a row of K and of V (what a row takes for itself, its scale and its place, is then for twice the values), `lanes` chunks apart.
// W: values of a chunk, 16 bytes, or 1 for rows that do not start on 16 bytes (chunks of four values, one by one)
constexpr int kChunks = 2;
template <typename T, int W> constexpr int kChunk = W > 1 ? W : 4;

// Row i of the block's rows: its token and head
__device__ __forceinline__ void row_at(const MoveArgs &a, int i, int &t, int &head)
{
    t = a.c.heads == 1 ? i : (int)__umulhi((uint32_t)i, a.per_head);
    head = i - t * a.c.heads;
}

template <typename T, int FMT, int W>
__global__ void __launch_bounds__(kThreads)
cache_write_kernel(const MoveArgs a)
{
    dependency_wait();
    dependents_may_start();
    __shared__ long long places[kMostTokens];
    const int t0 = blockIdx.x * a.tokens, D = a.c.D, lane = threadIdx.x & (a.lanes - 1);
    constexpr int N = kChunk<T, W>;
    const int all = a.tokens * a.c.heads << a.log_lanes;
    float x[2][kChunks][N];
    int t, head;
    // (every thread of the warp takes part in the shuffles: those without a row have zeros)
    auto fetch = [&](int i0) {
        row_at(a, i0 >> a.log_lanes, t, head);
        const bool here = i0 < all && t < a.c.T - t0;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const T *src = static_cast<const T *>(w ? a.v : a.k) + ((long long)t0 + t) * (w ? a.v_stride : a.k_stride) + head * D;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int d = (lane + c * a.lanes) * N;
#pragma unroll
                for (int e = 0; e < N; ++e) x[w][c][e] = 0.0f;
                if (here && d < D) {
                    if constexpr (W > 1) load_values<T, W>(src + d, x[w][c]);
                    else
#pragma unroll
                        for (int e = 0; e < N; ++e) x[w][c][e] = to_float(src[d + e]);
                }
            }
        }
    };
    fetch(threadIdx.x);                              // (on their way while the places are looked up)
    places_of(a, t0, places);
    for (int i0 = threadIdx.x; i0 - (int)threadIdx.x < all; i0 += kThreads) {
        if (i0 != (int)threadIdx.x) fetch(i0);
        long long row = i0 < all ? places[t] : -2;
        const bool mine = row >= 0;
        row += (long long)head << a.c.shift;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint8_t *base = const_cast<uint8_t *>(w ? a.c.v : a.c.k);
            if constexpr (FMT == HIPGPT_CACHE_PLAIN) {
                T *dst = reinterpret_cast<T *>(base) + row * D;
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const int d = (lane + c * a.lanes) * N;
                    if (mine && d < D) store_values<T, N>(dst + d, x[w][c]);
                }
            } else {
                uint32_t most = 0;
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
#pragma unroll
                    for (int e = 0; e < N; ++e) most = max(most, __float_as_uint(x[w][c][e]) & 0x7FFFFFFFu);
                most = row_max(most, a.lanes);
                const bool whole = most < 0x7F800000u;
                float inv, s = scale_of<FMT>(__uint_as_float(most), inv);
                uint8_t *dst = base + row * D;
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const int d = (lane + c * a.lanes) * N;
                    uint32_t code[N / 4];
#pragma unroll
                    for (int e = 0; e < N / 4; ++e) {
                        const float *y = x[w][c] + 4 * e;
                        if constexpr (FMT == HIPGPT_CACHE_E4M3) code[e] = e4m3_pair(y[0] * inv, y[1] * inv) | e4m3_pair(y[2] * inv, y[3] * inv) << 16;
                        else code[e] = int8_word(y, s, inv);
                        if (!whole) code[e] = 0u;
                    }
                    if (mine && d < D) {
                        if constexpr (N == 8) *reinterpret_cast<uint2 *>(dst + d) = make_uint2(code[0], code[1]);
                        else *reinterpret_cast<uint32_t *>(dst + d) = code[0];
                    }
                }
                if (mine && lane == 0) const_cast<float *>(w ? a.c.vs : a.c.ks)[row] = whole ? s : __uint_as_float(0x7FFFFFFFu);
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
    __shared__ long long places[kMostTokens];
    const int t0 = blockIdx.x * a.tokens, D = a.c.D, lane = threadIdx.x & (a.lanes - 1);
    places_of(a, t0, places);
    constexpr int N = kChunk<T, W>;
    const int all = a.tokens * a.c.heads << a.log_lanes;
    for (int i = threadIdx.x; i < all; i += kThreads) {
        int t, head;
        row_at(a, i >> a.log_lanes, t, head);
        const long long place = places[t], row = place + ((long long)head << a.c.shift);
        if (place == -2) continue;
        float x[2][kChunks][N], s[2] = {0.0f, 0.0f};
        uint32_t word[2][kChunks][2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint8_t *base = w ? a.c.v : a.c.k;
            if constexpr (FMT != HIPGPT_CACHE_PLAIN) if (place >= 0) s[w] = __ldg((w ? a.c.vs : a.c.ks) + row);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int d = (lane + c * a.lanes) * N;
                word[w][c][0] = word[w][c][1] = 0u;
#pragma unroll
                for (int e = 0; e < N; ++e) x[w][c][e] = 0.0f;
                if (place < 0 || d >= D) continue;
                if constexpr (FMT == HIPGPT_CACHE_PLAIN) {
                    load_values<T, N>(reinterpret_cast<const T *>(base) + row * D + d, x[w][c]);
                } else if constexpr (N == 8) {
                    const uint2 y = *reinterpret_cast<const uint2 *>(base + row * D + d);
                    word[w][c][0] = y.x; word[w][c][1] = y.y;
                } else {
                    word[w][c][0] = *reinterpret_cast<const uint32_t *>(base + row * D + d);
                }
            }
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            T *dst = static_cast<T *>(const_cast<void *>(w ? a.v : a.k)) + (t0 + t) * (w ? a.v_stride : a.k_stride) + head * D;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int d = (lane + c * a.lanes) * N;
                if (d >= D) continue;
                if constexpr (FMT != HIPGPT_CACHE_PLAIN)
#pragma unroll
                    for (int e = 0; e < N / 4; ++e) {
                        uint32_t lo, hi;
                        codes_to_half<FMT>(word[w][c][e], lo, hi);
                        const float2 a = floats_of(lo), b = floats_of(hi);
                        x[w][c][4 * e] = a.x * s[w];
                        x[w][c][4 * e + 1] = a.y * s[w];
                        x[w][c][4 * e + 2] = b.x * s[w];
                        x[w][c][4 * e + 3] = b.y * s[w];
                    }
                if constexpr (W > 1) store_values<T, W>(dst + d, x[w][c]);
                else
#pragma unroll
                    for (int e = 0; e < N; ++e) dst[d + e] = from_float<T>(x[w][c][e]);
            }
        }
    }
}

template <typename T, int FMT>
int launch_move(MoveArgs a, bool write, cudaStream_t st)
{
    constexpr int W = kPer16<T>;
    const bool vec = all_aligned16({a.k, a.v}) && a.k_stride % W == 0 && a.v_stride % W == 0;
    // As many threads as take D values two chunks each, rounded up to a power of two
    a.log_lanes = 0;
    while (kChunks * (vec ? W : 4) << a.log_lanes < a.c.D) ++a.log_lanes;
    a.lanes = 1 << a.log_lanes;
    // Tokens a block: one where there are few, 32 (whose places are looked up side by side) where there are enough for eight blocks an SM
    const long long each = (long long)a.c.heads << a.log_lanes;
    a.tokens = 1;
    while (a.tokens < kMostTokens && (a.tokens * each < kThreads || a.c.T / (2 * a.tokens) >= 148 * 8) && a.c.T >= 2 * a.tokens * 148) a.tokens *= 2;
    const long long blocks = ((long long)a.c.T + a.tokens - 1) / a.tokens;
    a.per_head = (uint32_t)(((1ull << 32) + a.c.heads - 1) / a.c.heads);             // (of one head: not used)
    if (each * a.tokens > 1LL << 30 || ((long long)a.tokens * a.c.heads + kThreads) * a.c.heads >= 1LL << 32) return fail(HIPGPT_ERR_BAD_ARG, "rows of %d heads are beyond one call", a.c.heads);
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
