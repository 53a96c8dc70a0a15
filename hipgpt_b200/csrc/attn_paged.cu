// Attention of new tokens over a paged cache, in registers: the kernel for single tokens and for fp32.
//
//   out = softmax(scale q K^T) V per row, one pass over the keys with the running maximum and sum
//
// Bound for single tokens: HBM, the cache is read once (the group's rows share it).  So K and V go from global memory straight to the registers of the warp that
// multiplies them (mma.sync: sixteen rows by eight keys; what tcgen05 adds is not needed where the bytes decide, and its operands would have to lie in
// shared memory first):
//   * which 16 values of a row an instruction sums over does not matter as long as Q's are the same, so a thread of the four that share a key takes 16
//     consecutive bytes of its row, and Q is laid out to match;
//   * P's layout as a result (keys 2t, 2t+1, 8+2t, 9+2t of sixteen) is its layout as an operand, so a thread takes 16 consecutive bytes of each of those four rows of V, and the
//     column of V^T that an instruction needs is one byte (or half) picked from each of two registers by the permutation that widening the codes takes anyway.
// Shared memory holds Q (a block's warps take the same rows and different keys) and the warps' results at the end.  Each warp has a block of V on its way while it works on
// K, and the next block of K while it works on V.
// Codes are widened to bf16 (exact); a key's scale multiplies its scores, a value's scale its probabilities.
// fp32 operands are three bf16 pieces (24 bits); products of pieces whose orders add up to more than two are left out.  The tensor core cuts off where others round, so no fp32 sum
// stays in it for more than a block of keys.
#include "attn_paged.cuh"
#include "stream_workspace.hpp"

#include <math.h>

namespace hipgpt {

StreamWorkspace g_paged_ws;                      // parts of tiles (attn_paged_tc.cu's too)

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;

// D += A B: 16 rows, 8 columns, 16 summed over; bf16
__device__ __forceinline__ void mma16(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// Piece i of N of two fp32 values as bf16 pairs; what is left in the values
__device__ __forceinline__ uint32_t next_piece(float &lo, float &hi)
{
    const uint32_t w = pack_bf16(lo, hi);
    lo -= __uint_as_float(w << 16);
    hi -= __uint_as_float(w & 0xFFFF0000u);
    return w;
}

template <int BYTES>
__device__ __forceinline__ void load_words(uint32_t *w, const uint8_t *p, bool there)
{
    if constexpr (BYTES == 16) {
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (there) u = __ldg(reinterpret_cast<const uint4 *>(p));
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (BYTES == 8) {
        uint2 u = make_uint2(0u, 0u);
        if (there) u = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = u.x; w[1] = u.y;
    } else {
        static_assert(BYTES == 4, "a word at least");
        w[0] = there ? __ldg(reinterpret_cast<const uint32_t *>(p)) : 0u;
    }
}

constexpr int least_of(int a, int b) { return a < b ? a : b; }

template <typename T, int FMT, int DP, bool SPLITROWS>
struct Shape {
    static constexpr bool F32 = sizeof(T) == 4, CODED = FMT != HIPGPT_CACHE_PLAIN;
    static constexpr int EB = CODED ? 1 : (int)sizeof(T);               // bytes of an element of the cache
    static constexpr int NQ = F32 ? 3 : 1, NK = F32 && !CODED ? 3 : 1;  // pieces of Q and P, of K and V
    static constexpr int MT = SPLITROWS && DP <= 64 ? 2 : 1;            // tiles of 16 rows a warp
    static constexpr int ROWS = 16 * MT * (SPLITROWS ? kWarps : 1);
    // keys a warp takes at a time: 32 registers of K and as many of V
    static constexpr int KB = 4096 / (DP * EB) >= 32 ? 32 : 16;
    static constexpr int UNIT = SPLITROWS ? 64 : kWarps * KB;
    static constexpr int EC = least_of(16 / EB, DP / 4), NC = DP / 4 / EC;       // K: elements of a chunk, chunks a thread
    static constexpr int EV = least_of(16 / EB, DP / 8), NV = DP / 8 / EV;       // V: the same
    static constexpr int STEPS = DP / 16, TILES = DP / 8;
    static constexpr size_t kQBytes = (size_t)NQ * (ROWS / 16) * STEPS * 32 * 16;
    static constexpr int kPad = DP + 4;
    static constexpr size_t kOBytes = SPLITROWS ? 0 : (size_t)kWarps * ROWS * kPad * 4;
    static constexpr size_t kSmem = kQBytes + kOBytes;
};

template <typename T, int FMT, int DP, bool SPLITROWS>
__global__ void __launch_bounds__(kThreads, SPLITROWS || (sizeof(T) == 4 && DP == 128) ? 2 : 3)
paged_rows_kernel(const AttnArgs a)
{
    using C = Shape<T, FMT, DP, SPLITROWS>;
    extern __shared__ __align__(16) uint8_t smem[];
    uint4 *q_s = reinterpret_cast<uint4 *>(smem);
    float *o_s = reinterpret_cast<float *>(smem + C::kQBytes);
    __shared__ long long sums[kWarps + 2];
    __shared__ float2 ml_s[kWarps][16];
    dependency_wait();
    dependents_may_start();

    const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int D = a.c.D;
    Run<C::ROWS, C::UNIT, kThreads> run(a);
    int4 cut = make_int4(0, 0, 0, -1);
    bool more = run.begin(sums);
    for (; more; more = run.next()) {
        const Tile w = run.at();
        const Sequence &s = w.s;
        const long long rows = (long long)s.n * a.group;
        const int row0 = w.tile * C::ROWS;

        // ---- Q as operands ----------------------------------------------------------------------------------------
        __syncthreads();                         // (the tile before has been read)
        for (int i = tid; i < (C::ROWS / 16) * C::STEPS * 32; i += kThreads) {
            const int l = i & 31, ks = (i >> 5) % C::STEPS, mt = (i >> 5) / C::STEPS;
            const int d = ((l & 3) + 4 * (ks / (C::EC / 4))) * C::EC + 4 * (ks % (C::EC / 4));
            float x[2][4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const long long row = row0 + mt * 16 + (l >> 2) + 8 * r;
                const bool there = row < rows && d < D;
                const T *src = static_cast<const T *>(a.q) + (s.first + row / a.group) * a.q_stride + (long long)(w.head * a.group + (int)(row % a.group)) * D + d;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[r][e] = there ? to_float(src[e]) : 0.0f;
            }
#pragma unroll
            for (int n = 0; n < C::NQ; ++n) {
                uint4 f;
                f.x = next_piece(x[0][0], x[0][1]);
                f.y = next_piece(x[1][0], x[1][1]);
                f.z = next_piece(x[0][2], x[0][3]);
                f.w = next_piece(x[1][2], x[1][3]);
                q_s[n * (C::ROWS / 16) * C::STEPS * 32 + i] = f;
            }
        }
        __syncthreads();
        const uint4 *q_w = q_s + (SPLITROWS ? warp * C::MT * C::STEPS * 32 : 0) + lane;

        int limit[C::MT][2];
        const int wrow = row0 + (SPLITROWS ? warp * 16 * C::MT : 0);
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) limit[mt][r] = limit_of(a, s, wrow + mt * 16 + g + 8 * r);
        const int least_limit = limit_of(a, s, wrow);
        const int keys = tile_keys<C::ROWS>(a, s, w.tile);
        const long long wlast = min((long long)wrow + 16 * C::MT, rows) - 1;             // this warp's rows end here, and their keys
        const int wkeys = !SPLITROWS ? keys : wlast < wrow ? 0 : limit_of(a, s, (int)wlast);

        float o[C::MT][C::TILES][4], m[C::MT][2], l[C::MT][2];
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
#pragma unroll
            for (int j = 0; j < C::TILES; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][j][e] = 0.0f;
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.0f;
        }

        // ---- blocks of KB keys ------------------------------------------------------------------------------------
        constexpr int NG = C::KB / 16, NJ = C::KB / 8, PER_UNIT = C::UNIT / C::KB, STEP = SPLITROWS ? 1 : kWarps;
        const int blk_end = min(w.to * PER_UNIT, (wkeys + C::KB - 1) / C::KB);
        uint32_t kreg[NJ][C::NC][C::EC * C::EB / 4], vreg[NG][4][C::NV][C::EV * C::EB / 4];
        float2 kscale[C::CODED ? NJ : 1], vscale[C::CODED ? NJ : 1];
        long long at[NG], next_at[NG];           // the first row of each 16 keys in the cache
        auto find = [&](long long (&where)[NG], int blk) {
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const int p = blk * C::KB + 16 * i;
                where[i] = blk < blk_end && p < wkeys ? row_of(a.c, w.b, w.head, p) : -1;
            }
        };
        auto load_k = [&](const long long (&where)[NG], int blk) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int in = 8 * (j & 1) + g;
                const bool there = where[j / 2] >= 0 && blk * C::KB + 16 * (j / 2) + in < wkeys;
                const uint8_t *row = a.c.k + (where[j / 2] + in) * D * C::EB;
#pragma unroll
                for (int i = 0; i < C::NC; ++i) {
                    const int d = (t4 + 4 * i) * C::EC;
                    load_words<C::EC * C::EB>(kreg[j][i], row + d * C::EB, there && d < D);
                }
                if constexpr (C::CODED) kscale[j] = where[j / 2] >= 0 ? __ldg(reinterpret_cast<const float2 *>(a.c.ks + where[j / 2] + 8 * (j & 1) + 2 * t4)) : make_float2(0.0f, 0.0f);
            }
        };
        auto load_v = [&](int blk) {
#pragma unroll
            for (int i = 0; i < NG; ++i) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int in = 8 * (x >> 1) + 2 * t4 + (x & 1);
                    const bool there = at[i] >= 0 && blk * C::KB + 16 * i + in < wkeys;
                    const uint8_t *row = a.c.v + (at[i] + in) * D * C::EB;
#pragma unroll
                    for (int c = 0; c < C::NV; ++c) {
                        const int d = (g + 8 * c) * C::EV;
                        load_words<C::EV * C::EB>(vreg[i][x][c], row + d * C::EB, there && d < D);
                    }
                }
            }
            if constexpr (C::CODED)
#pragma unroll
                for (int j = 0; j < NJ; ++j) vscale[j] = at[j / 2] >= 0 ? __ldg(reinterpret_cast<const float2 *>(a.c.vs + at[j / 2] + 8 * (j & 1) + 2 * t4)) : make_float2(0.0f, 0.0f);
        };
        const int blk0 = w.from * PER_UNIT + (SPLITROWS ? 0 : warp);
        find(at, blk0);
        load_k(at, blk0);
        for (int blk = blk0; blk < blk_end; blk += STEP) {
            load_v(blk);
            find(next_at, blk + STEP);
            // scores: the main products, and apart from them those of the smaller pieces
            float z[C::MT][NJ][4], zc[C::F32 ? C::MT : 1][C::F32 ? NJ : 1][4];
#pragma unroll
            for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        z[mt][j][e] = 0.0f;
                        if constexpr (C::F32) zc[mt][j][e] = 0.0f;
                    }
#pragma unroll
            for (int ks = 0; ks < C::STEPS; ++ks) {
                uint4 q[C::NQ][C::MT];
#pragma unroll
                for (int n = 0; n < C::NQ; ++n)
#pragma unroll
                    for (int mt = 0; mt < C::MT; ++mt) q[n][mt] = q_w[(n * (C::ROWS / 16) + mt) * C::STEPS * 32 + ks * 32];
                constexpr int PER = C::EC / 4;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const uint32_t *kw = kreg[j][ks / PER];
                    uint32_t b[C::NK][2];
                    if constexpr (C::CODED) {
                        const uint32_t x = kw[ks % PER];
                        b[0][0] = code_pair<FMT>(x, x, 0, 1);
                        b[0][1] = code_pair<FMT>(x, x, 2, 3);
                    } else if constexpr (!C::F32) {
                        b[0][0] = kw[2 * (ks % PER)];
                        b[0][1] = kw[2 * (ks % PER) + 1];
                    } else {
                        float x[4] = {__uint_as_float(kw[0]), __uint_as_float(kw[1]), __uint_as_float(kw[2]), __uint_as_float(kw[3])};
#pragma unroll
                        for (int n = 0; n < 3; ++n) {
                            b[n][0] = next_piece(x[0], x[1]);
                            b[n][1] = next_piece(x[2], x[3]);
                        }
                    }
#pragma unroll
                    for (int mt = 0; mt < C::MT; ++mt) {
                        if constexpr (C::F32) {
#pragma unroll
                            for (int order = 2; order >= 1; --order)
#pragma unroll
                                for (int n = 0; n <= order && n < C::NK; ++n) mma16(zc[mt][j], q[order - n][mt], b[n][0], b[n][1]);
                        }
                        mma16(z[mt][j], q[0][mt], b[0][0], b[0][1]);
                    }
                }
            }
            float2 ks2[C::CODED ? NJ : 1];
            if constexpr (C::CODED)
#pragma unroll
                for (int j = 0; j < NJ; ++j) ks2[j] = kscale[j];
            load_k(next_at, blk + STEP);

            // ---- softmax ----------------------------------------------------------------------------------------------
            const int p0 = blk * C::KB;
            bool masked = p0 + C::KB > least_limit;
#pragma unroll
            for (int i = 0; i < NG; ++i) masked = masked || at[i] < 0;
            uint4 p[C::NQ][C::MT][NG];
#pragma unroll
            for (int mt = 0; mt < C::MT; ++mt) {
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = z[mt][j][e];
                        if constexpr (C::F32) x += zc[mt][j][e];
                        if constexpr (C::CODED) x *= (e & 1) ? ks2[j].y : ks2[j].x;
                        x *= a.cscale;
                        if (masked && !(p0 + 8 * j + 2 * t4 + (e & 1) < limit[mt][e >> 1] && at[j / 2] >= 0)) x = -INFINITY;
                        z[mt][j][e] = x;
                        top[e >> 1] = fmaxf(top[e >> 1], x);
                    }
                float base[2], alpha[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                    const float now = fmaxf(m[mt][r], top[r]);
                    base[r] = now == -INFINITY ? 0.0f : now;
                    alpha[r] = ex2_approx(m[mt][r] - base[r]);
                    m[mt][r] = now;
                    l[mt][r] *= alpha[r];
                }
                if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                    for (int j = 0; j < C::TILES; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[mt][j][e] *= alpha[e >> 1];
                }
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = z[mt][j][e];
                        float y = ex2_approx(x - base[e >> 1]);
                        l[mt][e >> 1] += y;
                        if constexpr (C::CODED) {
                            y *= (e & 1) ? vscale[j].y : vscale[j].x;
                            if (masked && x == -INFINITY) y = 0.0f;              // (the scale of a place that holds nothing may be anything)
                        }
                        z[mt][j][e] = y;
                    }
#pragma unroll
                for (int i = 0; i < NG; ++i)
#pragma unroll
                    for (int n = 0; n < C::NQ; ++n) {
                        p[n][mt][i].x = next_piece(z[mt][2 * i][0], z[mt][2 * i][1]);
                        p[n][mt][i].y = next_piece(z[mt][2 * i][2], z[mt][2 * i][3]);
                        p[n][mt][i].z = next_piece(z[mt][2 * i + 1][0], z[mt][2 * i + 1][1]);
                        p[n][mt][i].w = next_piece(z[mt][2 * i + 1][2], z[mt][2 * i + 1][3]);
                    }
            }

            // ---- P V --------------------------------------------------------------------------------------------------
#pragma unroll
            for (int c = 0; c < C::NV; ++c)
#pragma unroll
                for (int e = 0; e < C::EV; ++e) {
                    const int j = c * C::EV + e;
                    uint32_t b[NG][C::NK][2];
#pragma unroll
                    for (int i = 0; i < NG; ++i)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            const uint32_t *w0 = vreg[i][2 * hf][c], *w1 = vreg[i][2 * hf + 1][c];
                            if constexpr (C::CODED) {
                                b[i][0][hf] = code_pair<FMT>(w0[e / 4], w1[e / 4], e & 3, e & 3);
                            } else if constexpr (!C::F32) {
                                b[i][0][hf] = __byte_perm(w0[e / 2], w1[e / 2], e & 1 ? 0x7632 : 0x5410);
                            } else {
                                float x = __uint_as_float(w0[e]), y = __uint_as_float(w1[e]);
#pragma unroll
                                for (int n = 0; n < 3; ++n) b[i][n][hf] = next_piece(x, y);
                            }
                        }
#pragma unroll
                    for (int mt = 0; mt < C::MT; ++mt) {
                        if constexpr (C::F32) {
                            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int order = 2; order >= 0; --order)
#pragma unroll
                                for (int n = 0; n <= order && n < C::NK; ++n)
#pragma unroll
                                    for (int i = 0; i < NG; ++i) mma16(d, p[order - n][mt][i], b[i][n][0], b[i][n][1]);
#pragma unroll
                            for (int x = 0; x < 4; ++x) o[mt][j][x] += d[x];
                        } else {
#pragma unroll
                            for (int i = 0; i < NG; ++i) mma16(o[mt][j], p[0][mt][i], b[i][0][0], b[i][0][1]);
                        }
                    }
                }
#pragma unroll
            for (int i = 0; i < NG; ++i) at[i] = next_at[i];
        }
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                l[mt][r] += __shfl_xor_sync(0xffffffffu, l[mt][r], 1);
                l[mt][r] += __shfl_xor_sync(0xffffffffu, l[mt][r], 2);
            }

        // ---- the tile's end ---------------------------------------------------------------------------------------
        const int part = run.part();
        if (part >= 0 && (part & 1)) cut = run.cut();
        float *dst = part < 0 ? nullptr : a.parts + (size_t)part * C::ROWS * (DP + 2);
        // columns of TILES' tile c * EV + e: values (2 t4 + 8 c) EV + e and (2 t4 + 1 + 8 c) EV + e
        if constexpr (!SPLITROWS) {
            // the warps' sums by way of shared memory; a warp joins four rows
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float *row = o_s + (warp * 16 + g + 8 * r) * C::kPad;
#pragma unroll
                for (int c = 0; c < C::NV; ++c)
#pragma unroll
                    for (int e = 0; e < C::EV; ++e) {
                        row[(2 * t4 + 8 * c) * C::EV + e] = o[0][c * C::EV + e][2 * r];
                        row[(2 * t4 + 1 + 8 * c) * C::EV + e] = o[0][c * C::EV + e][2 * r + 1];
                    }
                if (t4 == 0) ml_s[warp][g + 8 * r] = make_float2(m[0][r], l[0][r]);
            }
            __syncthreads();
            for (int r = warp; r < 16; r += kWarps) {
                const long long row = row0 + r;
                if (row >= rows) break;
                float top = -INFINITY, sum = 0.0f, f[kWarps];
#pragma unroll
                for (int x = 0; x < kWarps; ++x) top = fmaxf(top, ml_s[x][r].x);
                const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
                for (int x = 0; x < kWarps; ++x) {
                    f[x] = ex2_approx(ml_s[x][r].x - base);
                    sum = fmaf(ml_s[x][r].y, f[x], sum);
                }
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const long long t = s.first + row / a.group;
                T *out = static_cast<T *>(a.out) + t * a.out_stride + (long long)(w.head * a.group + (int)(row % a.group)) * D;
                bool wild = false;
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) {
                    const int d = lane + 32 * i;
                    float y = 0.0f;
#pragma unroll
                    for (int x = 0; x < kWarps; ++x) y = fmaf(o_s[(x * 16 + r) * C::kPad + d], f[x], y);
                    if (dst) {
                        dst[(size_t)r * DP + d] = y;
                    } else {
                        y = sum == 0.0f ? 0.0f : y * inv;
                        wild = wild || !(fabsf(y) <= 3.402823466e38f);
                        if (d < D) out[d] = from_float<T>(y);
                    }
                }
                if (dst) {
                    if (lane == 0) reinterpret_cast<float2 *>(dst + C::ROWS * DP)[r] = make_float2(top, sum);
                } else if (__any_sync(0xffffffffu, wild)) {
                    __syncwarp();
                    mend_row<T, FMT>(a, w.b, w.head, s, (int)row, keys);
                }
            }
        } else {
            bool wild[C::MT][2];
#pragma unroll
            for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    wild[mt][r] = false;
                    const int rr = (warp * C::MT + mt) * 16 + g + 8 * r;
                    const long long row = row0 + rr;
                    const float sum = l[mt][r], inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    const bool there = row < rows;
                    const long long t = s.first + row / a.group;
                    T *out = static_cast<T *>(a.out) + t * a.out_stride + (long long)(w.head * a.group + (int)(row % a.group)) * D;
#pragma unroll
                    for (int c = 0; c < C::NV; ++c)
#pragma unroll
                        for (int e = 0; e < C::EV; ++e)
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const int d = (2 * t4 + x + 8 * c) * C::EV + e;
                                const float y = o[mt][c * C::EV + e][2 * r + x];
                                if (dst) {
                                    if (there) dst[(size_t)rr * DP + d] = y;
                                } else {
                                    const float v = sum == 0.0f ? 0.0f : y * inv;
                                    wild[mt][r] = wild[mt][r] || (there && !(fabsf(v) <= 3.402823466e38f));
                                    if (there && d < D) out[d] = from_float<T>(v);
                                }
                            }
                    if (dst && there && t4 == 0) reinterpret_cast<float2 *>(dst + C::ROWS * DP)[rr] = make_float2(m[mt][r], sum);
                }
            if (!dst) {
#pragma unroll
                for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        unsigned some = __ballot_sync(0xffffffffu, wild[mt][r]);
                        __syncwarp();
                        while (some) {
                            const int who = (__ffs((int)some) - 1) >> 2;         // its row in the tile's eight
                            some &= ~(0xFu << (4 * who));
                            mend_row<T, FMT>(a, w.b, w.head, s, row0 + (warp * C::MT + mt) * 16 + who + 8 * r, keys);
                        }
                    }
            }
        }
    }
    if (a.cuts && tid == 0) {
        a.cuts[blockIdx.x] = cut;
        a.whole[blockIdx.x] = 1;
    }
}

template <typename T, int FMT, int DP, bool SPLITROWS>
int launch_rows(AttnArgs a, cudaStream_t st)
{
    using C = Shape<T, FMT, DP, SPLITROWS>;
    const auto kern = paged_rows_kernel<T, FMT, DP, SPLITROWS>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    static std::atomic<unsigned long long> done{0};
    static std::atomic<int> resident{0};         // blocks on all SMs at once (the same on every B200)
    if (e == cudaSuccess) e = once_per_device(done, dev, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem); });
    int grid = resident.load(std::memory_order_relaxed);
    if (e == cudaSuccess && grid == 0) {
        int per = 0, sms = 0;
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, kThreads, C::kSmem);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        if (e == cudaSuccess) resident.store(grid = per * sms, std::memory_order_relaxed);
    }
    if (e != cudaSuccess || grid <= 0) return fail(HIPGPT_ERR_CUDA, "paged attention: %s", cudaGetErrorString(e));
    // no more blocks than there can be units; where no tile can be cut, no parts
    const long long room = (long long)a.c.most_pages << a.c.shift;
    const long long most = (room + C::UNIT - 1) / C::UNIT > 1 ? (room + C::UNIT - 1) / C::UNIT : 1;      // units of a tile
    const long long tiles = ((long long)a.c.T * a.group / C::ROWS + (a.c.T < a.c.B ? a.c.T : a.c.B)) * a.c.heads;
    a.least = 1;
    if (tiles < (1LL << 40) / most && tiles * most < grid) grid = (int)(tiles * most);
    const bool cuts = most > 1;
    StreamWorkspace::Lease ws;
    if (cuts) {
        const size_t parts = (size_t)2 * grid * C::ROWS * (DP + 2) * sizeof(float);
        const int rc = g_paged_ws.enter(st, parts + (size_t)grid * (sizeof(int4) + sizeof(int)), &ws);
        if (rc != HIPGPT_OK) return rc;
        a.parts = reinterpret_cast<float *>(ws.get());
        a.cuts = reinterpret_cast<int4 *>(ws.get() + parts);
        a.whole = reinterpret_cast<int *>(a.cuts + grid);
    }
    e = launch_overlapped(kern, dim3((unsigned)grid), dim3(kThreads), C::kSmem, st, a);
    if (e == cudaSuccess && cuts) e = launch_overlapped(paged_join_kernel<T, FMT, C::ROWS, DP>, dim3((unsigned)grid, (unsigned)(C::ROWS + 15) / 16), dim3(256), 0, st, a);
    return e == cudaSuccess ? check_launch("paged_rows_kernel") : fail(HIPGPT_ERR_CUDA, "paged_rows_kernel: %s", cudaGetErrorString(e));
}

template <typename T, int FMT, bool SPLITROWS>
int launch_rows_of(const AttnArgs &a, cudaStream_t st)
{
    return a.c.D <= 32 ? launch_rows<T, FMT, 32, SPLITROWS>(a, st) : a.c.D <= 64 ? launch_rows<T, FMT, 64, SPLITROWS>(a, st) : launch_rows<T, FMT, 128, SPLITROWS>(a, st);
}

template <typename T>
int launch_paged(int format, const AttnArgs &a, cudaStream_t st)
{
    const bool few = (long long)a.c.T * a.group <= 32LL * a.c.B;
    if constexpr (sizeof(T) == 2) {
        if (!few && a.c.pages > 0) return launch_paged_tc(format, a, st);          // (without pages there is nothing to copy)
        return format == HIPGPT_CACHE_PLAIN ? launch_rows_of<T, HIPGPT_CACHE_PLAIN, false>(a, st)
             : format == HIPGPT_CACHE_E4M3  ? launch_rows_of<T, HIPGPT_CACHE_E4M3, false>(a, st) : launch_rows_of<T, HIPGPT_CACHE_INT8, false>(a, st);
    } else {
        if (format == HIPGPT_CACHE_PLAIN) return few ? launch_rows_of<T, HIPGPT_CACHE_PLAIN, false>(a, st) : launch_rows_of<T, HIPGPT_CACHE_PLAIN, true>(a, st);
        if (format == HIPGPT_CACHE_E4M3) return few ? launch_rows_of<T, HIPGPT_CACHE_E4M3, false>(a, st) : launch_rows_of<T, HIPGPT_CACHE_E4M3, true>(a, st);
        return few ? launch_rows_of<T, HIPGPT_CACHE_INT8, false>(a, st) : launch_rows_of<T, HIPGPT_CACHE_INT8, true>(a, st);
    }
}

}  // namespace

void paged_release_scratch() { g_paged_ws.release(); }

}  // namespace hipgpt

using namespace hipgpt;

extern "C" int hipgpt_paged_attention(const hipgpt_paged_cache *cache, const hipgpt_paged_batch *batch, const void *d_q, long long q_stride, void *d_out, long long out_stride,
                                      int H, int causal, float scale, void *stream)
{
    AttnArgs a = {};
    const int rc = check_paged(cache, batch, &a.c);
    if (rc < 0) return rc;
    if (H <= 0 || H % cache->heads || H / cache->heads > 1 << 16) return fail(HIPGPT_ERR_BAD_ARG, "%d query heads cannot share %d heads of the cache", H, cache->heads);
    if (!(scale > 0.0f && scale <= 3.402823466e38f)) return fail(HIPGPT_ERR_BAD_ARG, "scale = %g is not positive", (double)scale);
    const long long width = (long long)H * cache->head_dim;
    if (width > 1 << 24 || (long long)batch->tokens * (H / cache->heads) > 2147483647LL - 4096) return fail(HIPGPT_ERR_BAD_ARG, "%d tokens of %d heads are beyond one call", batch->tokens, H);
    if (rc > 0) return HIPGPT_OK;
    if (!d_q || !d_out) return fail(HIPGPT_ERR_NULL, "q and out must not be NULL");
    if (check_stride("q", q_stride, width) != HIPGPT_OK || check_stride("out", out_stride, width) != HIPGPT_OK) return HIPGPT_ERR_BAD_ARG;
    const size_t es = cache->type == HIPGPT_TYPE_F32 ? 4 : 2;
    const int over = refuse_rows_over({d_out, (size_t)out_stride * es, (size_t)width * es, batch->tokens}, {{d_q, (size_t)q_stride * es, (size_t)width * es, batch->tokens}}, cache, batch);
    if (over != HIPGPT_OK) return over;
    a.q = d_q; a.out = d_out;
    a.q_stride = q_stride; a.out_stride = out_stride;
    a.group = H / cache->heads;
    a.causal = causal != 0;
    a.scale = scale;
    a.cscale = scale * kLog2e;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return cache->type == HIPGPT_TYPE_F32 ? launch_paged<float>(cache->format, a, st) : launch_paged<__nv_bfloat16>(cache->format, a, st);
}
