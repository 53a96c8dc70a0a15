// Dropout whose mask is a function of a seed, a counter and the element's index, and is never stored: the backward pass is the
// same call on the gradient.  (The reference's dropout, hipgpt_dropout in layer_ops.cu, draws the same mask at every call.)
//
//   bits(i) = 16 of the 128 bits of Philox4x32-10 (J. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011) at the 128-bit
//             counter (offset + i / 8) under the 64-bit key `seed`: word (i % 8) / 2 of the four, its low half for even i
//   t       = floor(65536 p + 1/2), at most 65535
//   out(i)  = [residual(i) +] (bits(i) >= t ? in(i) * 65536 / (65536 - t) : 0)
//
// The scale belongs to the probability that is used (a multiple of 2^-16), so the expected value is the input's.  A dropped
// element is 0 whatever it held, NaN and infinities too.  fp32 arithmetic, rounded once.
//
// Bound: HBM (4 M fp32 values and more); for 16-bit values the generator's ten rounds, about 80 instructions for each counter, come near it: 5.4 TB/s at 67 M
// values without a residual, 6.4 TB/s with one, 6.8 TB/s for 33 M fp32 values with one.  16 bits a value, not 32, because that would be twice the rounds.
#include "elem_types.cuh"

namespace hipgpt {
namespace {

// Counters a thread: more 16-byte words on their way for it, which 16-bit values need (67 M of them: one 59.8 us, two 55.2, four 49.4; with a residual 68.6,
// 63.2, 63.1) and 32-bit ones do not (33 M with a residual: 59.3, 59.3, 60.0).  Fewer values are better spread over more blocks: one against four, 0.5 M 1.7 and 2.3 us, 4 M 4.4 and
// 5.5, 8 M 8.3 and 8.3, 16 M 16.2 and 14.4
template <typename T> constexpr int kPer = sizeof(T) == 2 ? 4 : 1;
constexpr long long kManyValues = 1 << 23;

struct Words { uint32_t w[4]; };

__device__ __forceinline__ Words philox(unsigned long long counter, unsigned long long seed)
{
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0;
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// One thread: PER counters, eight values each, 256 counters apart; all its values are asked for before the first counter is worked on.  in, residual and out may be
// one buffer: a thread reads what it writes.
template <typename T, bool RES, bool VEC, int PER>
__global__ void __launch_bounds__(256)
dropout_counter_kernel(const T *in, const T *res, T *out, unsigned long long seed, unsigned long long offset, const unsigned long long *counter,
                       uint32_t thr, float scale, long long n)
{
    dependency_wait();
    dependents_may_start();
    const long long first = (long long)blockIdx.x * (256 * PER) + threadIdx.x;
    if (first * 8 >= n) return;
    const unsigned long long base = offset + (counter ? *counter : 0ull);
    float x[PER][8], y[PER][8];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const long long i0 = (first + 256 * u) * 8;
        if (VEC && i0 + 8 <= n) {
            load_values<T, 8>(in + i0, x[u]);
            if constexpr (RES) load_values<T, 8>(res + i0, y[u]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[u][j] = i0 + j < n ? to_float(in[i0 + j]) : 0.0f;
                if constexpr (RES) y[u][j] = i0 + j < n ? to_float(res[i0 + j]) : 0.0f;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const long long i0 = (first + 256 * u) * 8;
        if (i0 >= n) return;
        const Words r = philox(base + (unsigned long long)(first + 256 * u), seed);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t bits = j & 1 ? r.w[j / 2] >> 16 : r.w[j / 2] & 0xFFFFu;
            x[u][j] = bits >= thr ? __fmul_rn(x[u][j], scale) : 0.0f;
            if constexpr (RES) x[u][j] = __fadd_rn(y[u][j], x[u][j]);
        }
        if (VEC && i0 + 8 <= n) {
            store_values<T, 8>(out + i0, x[u]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) if (i0 + j < n) out[i0 + j] = from_float<T>(x[u][j]);
        }
    }
}

template <typename T>
int launch_dropout_counter(const void *in, const void *res, void *out, unsigned long long seed, unsigned long long offset, const unsigned long long *counter,
                           uint32_t thr, long long n, cudaStream_t st)
{
    const bool vec = all_aligned16({in, res, out});
    constexpr int PER = kPer<T>;
    const bool few = n < kManyValues;
    const auto kern = !vec ? (res ? dropout_counter_kernel<T, true, false, 1> : dropout_counter_kernel<T, false, false, 1>)
                      : few ? (res ? dropout_counter_kernel<T, true, true, 1> : dropout_counter_kernel<T, false, true, 1>)
                            : (res ? dropout_counter_kernel<T, true, true, PER> : dropout_counter_kernel<T, false, true, PER>);
    const long long block = 2048LL * (!vec || few ? 1 : PER), blocks = (n + block - 1) / block;
    const cudaError_t e = launch_overlapped(kern, dim3((unsigned)blocks), dim3(256), 0, st, static_cast<const T *>(in), static_cast<const T *>(res), static_cast<T *>(out),
                                            seed, offset, counter, thr, 65536.0f / (float)(65536u - thr), n);
    return e == cudaSuccess ? check_launch("dropout_counter_kernel") : fail(HIPGPT_ERR_CUDA, "dropout_counter_kernel: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace hipgpt

using namespace hipgpt;

extern "C" int hipgpt_dropout_counter(const void *d_in, const void *d_residual, void *d_out, float p, unsigned long long seed, unsigned long long offset,
                                      const unsigned long long *d_counter, long long n, int type, void *stream)
{
    if (type != HIPGPT_TYPE_F32 && type != HIPGPT_TYPE_BF16) return fail(HIPGPT_ERR_BAD_ARG, "unknown type %d", type);
    if (!(p >= 0.0f && p < 1.0f)) return fail(HIPGPT_ERR_BAD_ARG, "p = %g is outside [0, 1)", (double)p);
    if (n < 0 || n > 1ll << 41) return fail(HIPGPT_ERR_BAD_ARG, "bad size: n=%lld", n);
    if (n == 0) return HIPGPT_OK;
    if (!d_in || !d_out) return fail(HIPGPT_ERR_NULL, "in and out must not be NULL");
    const size_t bytes = (size_t)n * (type == HIPGPT_TYPE_F32 ? 4 : 2);
    for (const void *src : {d_in, d_residual})
        if (src && src != d_out && ranges_overlap(src, bytes, d_out, bytes)) return fail(HIPGPT_ERR_BAD_ARG, "out overlaps an input without being it");
    if (d_counter && ranges_overlap(d_counter, sizeof(*d_counter), d_out, bytes)) return fail(HIPGPT_ERR_BAD_ARG, "out overlaps the counter");
    double t = (double)p * 65536.0 + 0.5;                // (exact: p has 24 bits)
    const uint32_t thr = t >= 65535.0 ? 65535u : (uint32_t)t;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return type == HIPGPT_TYPE_F32 ? launch_dropout_counter<float>(d_in, d_residual, d_out, seed, offset, d_counter, thr, n, st)
                                   : launch_dropout_counter<__nv_bfloat16>(d_in, d_residual, d_out, seed, offset, d_counter, thr, n, st);
}
