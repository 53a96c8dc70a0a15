// Rotary positions: the first R values of each head as R / 2 pairs, pair i turned by position * frequency i.
//
//   (a, b) -> magnitude * (a cos - b sin, a sin + b cos), backwards (the transpose, which is the gradient) with -sin
//
// A frequency comes as a 64-bit fraction of a turn, so position * frequency modulo a turn is one integer product, exact for any position; its signed value, in half
// turns, is rounded to fp32 once (2^-24 of the angle) and sincospi takes it.  In fp32 radians a position of 10^6 would leave 2^-5 of a radian.
//
// Bound: HBM, one read and one write of the heads; a thread keeps the sines and cosines of its pairs for as many heads as the grid can spare (kThreadsWanted), because for each head
// anew they would be about as many instructions as an SM has for the bytes.  32768 tokens, 40 heads of 128, bf16: 107 us, 6.3 TB/s; 16 heads of 64, half turned, fp32: 45 us, 6.0 TB/s (119 and 62 us with a head's
// loads behind the stores of the head before); 8 tokens of 16 heads of 32: 3.5 us.
#include "paged.cuh"

#include <math.h>

#include <cmath>

namespace hipgpt {
namespace {

struct RotaryArgs {
    const void *x;
    void *out;
    const int *positions;
    const unsigned long long *words;
    long long x_stride, out_stride;
    float magnitude;
    int T, H, D, R, lanes, heads_per;    // lanes: threads a token (turning, then copying), heads_per: heads a thread
};

// W values at a time, the same of both halves (HALVES) or W / 2 neighbouring pairs.  Lanes of a token: R / 2 / W (halves; W pairs each) or R / W that turn, then (D - R) / W that copy.
template <typename T, int W, bool HALVES>
__global__ void __launch_bounds__(256)
rotary_kernel(const RotaryArgs a, bool inverse)
{
    dependency_wait();
    dependents_may_start();
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long t = at / a.lanes;
    const int lane = (int)(at - t * a.lanes);
    if (t >= a.T) return;
    const int h0 = blockIdx.y * a.heads_per, h1 = min(a.H, h0 + a.heads_per);
    const T *x = static_cast<const T *>(a.x) + t * a.x_stride;
    T *out = static_cast<T *>(a.out) + t * a.out_stride;
    constexpr int PAIRS = HALVES ? W : (W > 1 ? W / 2 : 1);            // (W == 1: one pair, value by value)
    const int turning = a.R / 2 / PAIRS;
    // (U heads at a time: the next loads must not wait for these stores, and the compiler cannot know that x and out, which may be one, have no element of two heads in common)
    constexpr int U = 4;
    if (lane >= turning) {
        const int d = a.R + (lane - turning) * W;
        for (int h = h0; h < h1; h += U) {
            float v[U][W];
#pragma unroll
            for (int u = 0; u < U; ++u) if (h + u < h1) load_values<T, W>(x + (h + u) * a.D + d, v[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) if (h + u < h1) store_values<T, W>(out + (h + u) * a.D + d, v[u]);
        }
        return;
    }
    const int pos = __ldg(a.positions + t);
    float c[PAIRS], s[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        const long long phase = (long long)(__ldg(a.words + lane * PAIRS + i) * (unsigned long long)(long long)pos);
        sincospif(__ll2float_rn(phase) * 0x1p-63f, &s[i], &c[i]);
        c[i] *= a.magnitude;
        s[i] *= inverse ? -a.magnitude : a.magnitude;
    }
    auto turn = [&](int i, float p, float q, float &p2, float &q2) {
        p2 = fmaf(p, c[i], -(q * s[i]));
        q2 = fmaf(p, s[i], q * c[i]);
    };
    if constexpr (HALVES) {
        const int d = lane * W, e = d + a.R / 2;
        if constexpr (W > 1) {
            uint4 p4[U], q4[U];
            for (int h = h0; h < h1; h += U) {
#pragma unroll
                for (int u = 0; u < U; ++u) if (h + u < h1) {
                    p4[u] = *reinterpret_cast<const uint4 *>(x + (h + u) * a.D + d);
                    q4[u] = *reinterpret_cast<const uint4 *>(x + (h + u) * a.D + e);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) if (h + u < h1) {
                    float p[W], q[W];
                    unpack(p4[u], p, T());
                    unpack(q4[u], q, T());
#pragma unroll
                    for (int i = 0; i < W; ++i) turn(i, p[i], q[i], p[i], q[i]);
                    store_values<T, W>(out + (h + u) * a.D + d, p);
                    store_values<T, W>(out + (h + u) * a.D + e, q);
                }
            }
        } else {
            for (int h = h0; h < h1; ++h) {
                float p = to_float(x[h * a.D + d]), q = to_float(x[h * a.D + e]);
                turn(0, p, q, p, q);
                out[h * a.D + d] = from_float<T>(p);
                out[h * a.D + e] = from_float<T>(q);
            }
        }
    } else {
        const int d = lane * PAIRS * 2;
        constexpr int V = W > 1 ? W : 2;             // values of a head
        for (int h = h0; h < h1; h += U) {
            float v[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) if (h + u < h1) {
                if constexpr (W > 1) load_values<T, W>(x + (h + u) * a.D + d, v[u]);
                else for (int i = 0; i < 2; ++i) v[u][i] = to_float(x[(h + u) * a.D + d + i]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) if (h + u < h1) {
#pragma unroll
                for (int i = 0; i < PAIRS; ++i) turn(i, v[u][2 * i], v[u][2 * i + 1], v[u][2 * i], v[u][2 * i + 1]);
                if constexpr (W > 1) store_values<T, W>(out + (h + u) * a.D + d, v[u]);
                else for (int i = 0; i < 2; ++i) out[(h + u) * a.D + d + i] = from_float<T>(v[u][i]);
            }
        }
    }
}

constexpr long long kThreadsWanted = 148 * 2048;

template <typename T>
int launch_rotary(RotaryArgs a, int interleaved, bool inverse, cudaStream_t st)
{
    constexpr int W = kPer16<T>;
    // 16 bytes at a time where every part of every row starts on 16 bytes and is made of them
    const bool vec = all_aligned16({a.x, a.out}) && a.x_stride % W == 0 && a.out_stride % W == 0 && a.D % W == 0 && a.R % W == 0 && (interleaved || a.R / 2 % W == 0);
    const int w = vec ? W : 1;
    const bool copies = a.x != a.out;            // in place the others stay where they are
    a.lanes = (interleaved ? (vec ? a.R / W : a.R / 2) : a.R / 2 / w) + (copies ? (a.D - a.R) / w : 0);
    const long long threads = (long long)a.T * a.lanes;
    if (threads == 0) return HIPGPT_OK;
    // heads a thread: as many as leave kThreadsWanted of them
    long long parts = (kThreadsWanted + threads - 1) / threads;
    if (parts > a.H) parts = a.H;
    if (parts > 65535) parts = 65535;
    a.heads_per = (int)((a.H + parts - 1) / parts);
    parts = (a.H + a.heads_per - 1) / a.heads_per;
    const long long blocks = (threads + 255) / 256;
    if (blocks > 2147483647LL || parts > 65535) return fail(HIPGPT_ERR_BAD_ARG, "rotary: %d tokens of %d heads are beyond one call", a.T, a.H);
    const auto kern = interleaved ? (vec ? rotary_kernel<T, W, false> : rotary_kernel<T, 1, false>) : (vec ? rotary_kernel<T, W, true> : rotary_kernel<T, 1, true>);
    const cudaError_t e = launch_overlapped(kern, dim3((unsigned)blocks, (unsigned)parts), dim3(256), 0, st, a, inverse);
    return e == cudaSuccess ? check_launch("rotary_kernel") : fail(HIPGPT_ERR_CUDA, "rotary_kernel: %s", cudaGetErrorString(e));
}

constexpr double kTwoPi = 6.283185307179586476925286766559;

}  // namespace
}  // namespace hipgpt

using namespace hipgpt;

extern "C" int hipgpt_rotary_frequencies(double *h_freq, int R, double base, int scaling, double factor, double original, double low, double high)
{
    if (R < 0 || R % 2) return fail(HIPGPT_ERR_BAD_ARG, "R = %d is not an even number of values", R);
    if (!(base > 0.0) || !std::isfinite(base)) return fail(HIPGPT_ERR_BAD_ARG, "base = %g is not positive", base);
    if (scaling < HIPGPT_ROTARY_UNSCALED || scaling > HIPGPT_ROTARY_RAMP) return fail(HIPGPT_ERR_BAD_ARG, "unknown scaling %d", scaling);
    if (scaling != HIPGPT_ROTARY_UNSCALED && (!(factor > 0.0) || !std::isfinite(factor))) return fail(HIPGPT_ERR_BAD_ARG, "factor = %g is not positive", factor);
    if (scaling == HIPGPT_ROTARY_RAMP && (!(original > 0.0) || !(low < high) || !std::isfinite(original) || !std::isfinite(low) || !std::isfinite(high)))
        return fail(HIPGPT_ERR_BAD_ARG, "bad ramp: original=%g low=%g high=%g", original, low, high);
    if (R == 0) return HIPGPT_OK;
    if (!h_freq) return fail(HIPGPT_ERR_NULL, "freq must not be NULL");
    if (scaling == HIPGPT_ROTARY_BASE && R > 2) base *= pow(factor, (double)R / (R - 2));
    for (int i = 0; i < R / 2; ++i) {
        double f = pow(base, -2.0 * i / R);
        if (scaling == HIPGPT_ROTARY_LINEAR) f /= factor;
        if (scaling == HIPGPT_ROTARY_RAMP) {
            double keep = (original * f / kTwoPi - low) / (high - low);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
            f *= keep + (1.0 - keep) / factor;
        }
        h_freq[i] = f;
    }
    return HIPGPT_OK;
}

extern "C" int hipgpt_rotary_words(const double *h_freq, unsigned long long *h_words, int n)
{
    if (n < 0) return fail(HIPGPT_ERR_BAD_ARG, "bad size: n=%d", n);
    if (n == 0) return HIPGPT_OK;
    if (!h_freq || !h_words) return fail(HIPGPT_ERR_NULL, "freq and words must not be NULL");
    for (int i = 0; i < n; ++i) {
        if (!std::isfinite(h_freq[i])) return fail(HIPGPT_ERR_BAD_ARG, "frequency %d is not finite", i);
        const double turns = h_freq[i] / kTwoPi;
        const double part = turns - floor(turns);                       // [0, 1]: a whole turn is none
        const double scaled = ldexp(part, 64);
        h_words[i] = scaled >= 0x1p64 ? 0ull : (unsigned long long)scaled;
    }
    return HIPGPT_OK;
}

extern "C" int hipgpt_rotary(const void *d_x, long long x_stride, const int *d_positions, const unsigned long long *d_words, void *d_out, long long out_stride,
                             float magnitude, int interleaved, int inverse, int T, int H, int D, int R, int type, void *stream)
{
    if (type != HIPGPT_TYPE_F32 && type != HIPGPT_TYPE_BF16) return fail(HIPGPT_ERR_BAD_ARG, "unknown type %d", type);
    if (T < 0 || H < 0 || D < 0 || D > 1024 || R < 0 || R % 2 || R > D) return fail(HIPGPT_ERR_BAD_ARG, "bad size: T=%d H=%d D=%d R=%d", T, H, D, R);
    const long long width = (long long)H * D;
    if (width > 1 << 24) return fail(HIPGPT_ERR_BAD_ARG, "rows of %d heads of %d values are too long", H, D);
    if (T == 0 || width == 0) return HIPGPT_OK;
    if (!d_x || !d_out || (R > 0 && (!d_positions || !d_words))) return fail(HIPGPT_ERR_NULL, "x, positions, words and out must not be NULL");
    for (const long long s : {x_stride, out_stride})
        if (s < width || s > 1LL << 40) return fail(HIPGPT_ERR_BAD_ARG, "rotary: rows of %lld values cannot be %lld apart", width, s);
    const size_t es = type == HIPGPT_TYPE_F32 ? 4 : 2;
    const Rows out{d_out, (size_t)out_stride * es, (size_t)width * es, T}, x{d_x, (size_t)x_stride * es, (size_t)width * es, T};
    if (!(d_x == d_out && x_stride == out_stride) && rows_overlap(out, x)) return fail(HIPGPT_ERR_BAD_ARG, "out overlaps x without being it");
    if (R > 0 && (ranges_overlap(d_out, extent_of(out), d_positions, 4 * (size_t)T) || ranges_overlap(d_out, extent_of(out), d_words, 4 * (size_t)R)))
        return fail(HIPGPT_ERR_BAD_ARG, "out overlaps the positions or the frequencies");
    const RotaryArgs a = {d_x, d_out, d_positions, d_words, x_stride, out_stride, magnitude, T, H, D, R, 0, 0};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return type == HIPGPT_TYPE_F32 ? launch_rotary<float>(a, interleaved, inverse != 0, st) : launch_rotary<__nv_bfloat16>(a, interleaved, inverse != 0, st);
}
