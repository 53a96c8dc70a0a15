// Attention of new tokens over a paged cache on mma.sync: the kernel for single tokens and for fp32.
//
//   out = softmax(scale q K^T) V per row, one pass over the keys with the running maximum and sum
//
// Bound for single tokens: HBM, the cache is read once (the group's rows share it).  One warp brings K and V as they lie in their pages into a ring in shared memory by bulk copies, a lane a
// run of keys in one page; four warps multiply (sixteen rows by eight keys an instruction; what tcgen05 adds is not needed where the bytes decide, and its operands would have to be
// laid out once more).  (32 sequences of 8192 to 32768 tokens, 8 heads of 128 codes: loads straight into registers
// 641 us, 2.2 TB/s, too few bytes on their way; copies 316 us; with the products the other way round, below, 244; without the kernel's arguments copied to
// every thread's stack 227 us, 6.2 TB/s, and 253 in long runs.)
//   * which 16 values of a row an instruction sums over does not matter as long as Q's are the same, so a thread of the four that share a key takes 16
//     consecutive bytes of its row, and Q is laid out to match;
//   * P's layout as a result (keys 2t, 2t+1, 8+2t, 9+2t of sixteen) is its layout as an operand, so a thread takes 16 consecutive bytes of each of those four rows of V, and the
//     column of V^T that an instruction needs is one byte (or half) picked from each of two registers.
// Codes become fp16 (exact), and so does Q, a power of two for each row; a key's scale multiplies its scores, a value's scale its probabilities, all of one power of two that follows the largest.
// fp32 operands are two fp16 pieces (22 bits) against codes, three bf16 pieces (24 bits) against each other, without the products whose orders add up to more than two.  The tensor core cuts off
// where others round, so no sum stays in it for more than a block of keys, or (kKeptUnits) for too many of them.
#include "attn_paged.cuh"
#include "stream_workspace.hpp"

#include <math.h>

namespace hipgpt {

StreamWorkspace g_paged_ws;                      // parts of tiles (attn_paged_tc.cu's too)

namespace {

constexpr int kWarps = 4, kThreads = 32 * (kWarps + 1);

__device__ int g_rows_status = 0;
// The tensor core cuts sums off towards zero, about 2^-24 of a sum for each sixteen keys.  Where they stay in it from one block of keys to the next (single tokens), they are put aside after this many units: 8192
// keys of a warp at most, so 2^-15.
constexpr int kKeptUnits = 256;

// D += A B: 16 rows, 8 columns, 16 summed over; fp16 or bf16
template <bool HALF>
__device__ __forceinline__ void mma16(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1)
{
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
    else asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// The next piece of two fp32 values; what is left in the values.  bf16: a piece that others follow stays finite (values from 3.396e38 on would round to infinity, and nothing but NaN would be left),
// so an infinity goes on to the last.
template <bool HALF>
__device__ __forceinline__ uint32_t next_piece(float &lo, float &hi, bool last)
{
    if constexpr (HALF) {
        const uint32_t w = half2_of(lo, hi);
        const float2 f = floats_of(w);
        lo -= f.x;
        hi -= f.y;
        return w;
    } else {
        uint32_t w;
        if (last) w = pack_bf16(lo, hi);
        else asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
        lo -= __uint_as_float(w << 16);
        hi -= __uint_as_float(w & 0xFFFF0000u);
        return w;
    }
}

template <int BYTES>
__device__ __forceinline__ void read_words(uint32_t *w, const uint8_t *p)
{
    if constexpr (BYTES == 16) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (BYTES == 8) {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        w[0] = u.x; w[1] = u.y;
    } else {
        static_assert(BYTES == 4, "a word at least");
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}

__host__ __device__ constexpr int least_of(int a, int b) { return a < b ? a : b; }
__host__ __device__ constexpr int most_of(int a, int b) { return a > b ? a : b; }

// CUT: K and V come as pieces that were cut before the kernel
template <typename T, int FMT, int DP, bool SPLITROWS, bool CUT_ = false>
struct Shape {
    static constexpr bool F32 = sizeof(T) == 4, CODED = FMT != HIPGPT_CACHE_PLAIN, CUT = CUT_;
    static constexpr int EB = CODED ? 1 : (int)sizeof(T);               // bytes of an element of the cache
    static constexpr int NQ = !F32 ? 1 : CODED ? 2 : 3, NK = F32 && !CODED ? 3 : 1;  // pieces of Q and P, of K and V
    static constexpr int ROWS = 16 * (SPLITROWS ? kWarps : 1);
    static constexpr int KB = 4096 / (DP * EB) >= 32 ? 32 : 16;         // keys a warp takes at a time
    static constexpr int UNIT = CUT && DP > 32 ? 32 : SPLITROWS ? 64 : kWarps * KB;      // keys of a place in the ring
    static constexpr int EC = least_of(16 / EB, DP / 4), NC = DP / 4 / EC;       // K: elements of a chunk, chunks a thread
    static constexpr int EV = least_of(16 / EB, DP / 8), NV = DP / 8 / EV;       // V: the same
    static constexpr int STEPS = DP / 16, TILES = DP / 8;
    static constexpr int kQBytes = NQ * (ROWS / 16) * STEPS * 32 * 16;
    static constexpr int kPad = DP + 4;
    static constexpr int kOBytes = SPLITROWS ? 0 : 2 * 16 * kPad * 4;   // two warps' results
    static constexpr int kSlotBytes = UNIT * DP * (CUT ? 6 : EB) + (CODED ? UNIT * 4 : 0);
    static constexpr int kFixed = kQBytes + kOBytes + 1024;
    // places of the ring: four at least
    static constexpr int kBudget = (DP == 128 ? 112 : 74) * 1024;       // two or three blocks an SM
    static constexpr int kSlots = most_of(4, least_of(12, (kBudget - kFixed) / kSlotBytes));
    static constexpr size_t kSmem = (size_t)kQBytes + kOBytes + (size_t)kSlots * kSlotBytes;
    static constexpr int kBlocks = kSmem > 112 * 1024 ? 1 : DP == 128 || kSmem > 74 * 1024 ? 2 : 3;           // an SM
};

// The warp that asks for the copies: a place of the ring takes UNIT keys or values as they lie in their pages, then their scales; a lane a run of keys in one page
template <typename C, int THREADS, typename Wait>
__device__ __forceinline__ void bring(const AttnArgs &a, Run<C::ROWS, C::UNIT, THREADS> &run, bool more, uint8_t *ring, uint64_t *full, uint64_t *empty, uint32_t *there_s, Wait wait)
{
    const int lane = threadIdx.x & 31, D = a.c.D;
    uint32_t slot = 0;
    const int page_keys = 1 << a.c.shift, run_keys = min(page_keys, C::UNIT), runs = C::UNIT / run_keys;
    bool alive = true;
    for (; more; more = run.next()) {
        const Tile w = run.at();
        const int keys = tile_keys<C::ROWS>(a, w.s, w.tile);
        auto look = [&](int u) {                     // a page for each run of keys, asked for a unit ahead
            const int p = u * C::UNIT + lane * run_keys;
            const int pg = lane < runs && p < keys ? __ldg(a.c.table + (size_t)w.b * a.c.most_pages + (p >> a.c.shift)) : -1;
            return pg < a.c.pages ? pg : -1;
        };
        int page = look(w.from);
        for (int u = w.from; u < w.to; ++u) {
            const int p = u * C::UNIT + lane * run_keys;
            const int count = page >= 0 ? min(run_keys, keys - p) : 0, scales = C::CODED ? (count + 3) & ~3 : 0;         // (whole 16 bytes of scales)
            const long long row = ((((long long)page * a.c.heads) + w.head) << a.c.shift) + (p & (page_keys - 1));
            int bytes = count * D * C::EB + scales * 4;
            if constexpr (C::CUT) {
                bytes = C::kSlotBytes;
            } else {
#pragma unroll
                for (int o = 16; o; o >>= 1) bytes += __shfl_xor_sync(0xffffffffu, bytes, o);
            }
            // one bit for each sixteen keys
            const uint32_t some = __ballot_sync(0xffffffffu, page >= 0);
            uint32_t there = 0;
#pragma unroll
            for (int i = 0; i < C::UNIT / 16; ++i) there |= (some >> (16 * i / run_keys) & 1u) << i;
            page = u + 1 < w.to ? look(u + 1) : -1;
#pragma unroll
            for (int which = 0; which < 2; ++which, ++slot) {
                const int sl = slot % C::kSlots;
                if (slot >= C::kSlots) alive = wait(&empty[sl], ((slot / C::kSlots) & 1) ^ 1, 12) && alive;
                alive = __all_sync(0xffffffffu, alive);
                if (lane == 0 && alive) {
                    there_s[sl] = there;
                    mbar_arrive_expect_tx(&full[sl], (uint32_t)bytes);
                }
                __syncwarp();
                if constexpr (C::CUT) {
                    const long long place = ((long long)w.b * a.c.heads + w.head) * a.cut_units + u;
                    if (lane == 0 && alive) bulk_load(ring + sl * C::kSlotBytes, (which ? a.cut_v : a.cut_k) + place * C::kSlotBytes, C::kSlotBytes, &full[sl]);
                } else if (count > 0 && alive) {
                    uint8_t *dst = ring + sl * C::kSlotBytes;
                    bulk_load(dst + lane * run_keys * D * C::EB, (which ? a.c.v : a.c.k) + row * D * C::EB, (uint32_t)(count * D * C::EB), &full[sl]);
                    if constexpr (C::CODED) bulk_load(dst + C::UNIT * C::STEPS * 16 + lane * run_keys * 4, (which ? a.c.vs : a.c.ks) + row, (uint32_t)(scales * 4), &full[sl]);
                }
            }
        }
    }
}

template <typename T, int FMT, int DP, bool SPLITROWS, bool CUT = false>
__global__ void __launch_bounds__(kThreads, Shape<T, FMT, DP, SPLITROWS, CUT>::kBlocks)
paged_rows_kernel(const __grid_constant__ AttnArgs a)
{
    using C = Shape<T, FMT, DP, SPLITROWS, CUT>;
    constexpr bool HALF = C::CODED;
    constexpr int SLOTS = C::kSlots;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;                            // [slot][UNIT keys][D] as in the pages, then their scales
    uint4 *q_s = reinterpret_cast<uint4 *>(smem + SLOTS * C::kSlotBytes);
    float *o_s = reinterpret_cast<float *>(smem + SLOTS * C::kSlotBytes + C::kQBytes);
    __shared__ uint64_t full[SLOTS], empty[SLOTS];
    __shared__ uint32_t there_s[SLOTS];              // whether each 16 keys of a place have a page
    __shared__ long long sums[kWarps + 3];
    __shared__ float2 ml_s[2][16];
    __shared__ float q_unit[C::ROWS];
    __shared__ volatile int abort_flag;
    __shared__ uint32_t mend_s;                      // tiles of the run (their numbers modulo 32) with rows to look at again
    __shared__ typename Run<C::ROWS, C::UNIT, kThreads>::Start start_s;
    __shared__ int tops[kWarps];

    const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int D = a.c.D;
    if (tid == 0) {
        abort_flag = 0;
        mend_s = 0;
        for (int i = 0; i < SLOTS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kWarps);
        }
    }
    __syncthreads();
    dependency_wait();
    dependents_may_start();

    // sites: 11 keys or values landed, 12 place free
    auto wait = [&](uint64_t *bar, uint32_t parity, int site) {
        const bool over = a.expire != 0 && expires_now(a.expire, site);
        if (!over && mbar_test(bar, parity)) return true;
        if (!abort_flag) {
            if (!over && mbar_wait(bar, parity)) return true;
            abort_flag = 1;
            atomicCAS(&g_rows_status, 0, site);
            linger();
        }
        return false;
    };
    Run<C::ROWS, C::UNIT, kThreads> run(a);
    bool more = run.begin(sums);
    if (more) run.keep(&start_s);

    if (warp == kWarps) {
        bring<C, kThreads>(a, run, more, ring, full, empty, there_s, wait);
        __syncwarp();
        if (abort_flag) linger();
        return;
    }

    // ===================== the products =====================================================================
    auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); };       // of the four warps
    auto leave = [&](int sl) {
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&empty[sl])) : "memory");
    };
    uint32_t slot = 0, number = 0;                   // of places; of the tile in the run
    int4 cut = make_int4(0, 0, 0, -1);
    for (; more; more = run.next(), ++number) {
        const Tile w = run.at();
        const Sequence &s = w.s;
        const int rows = (int)min((long long)s.n * a.group, 2147483647LL);
        const int row0 = w.tile * C::ROWS;

        // ---- Q as operands ----------------------------------------------------------------------------------------
        meet();                                      // (the tile before has been read)
        if constexpr (HALF) {
            // a power of two for each row brings its largest value to [2^14, 2^15)
            for (int r = warp; r < C::ROWS; r += kWarps) {
                const int row = row0 + r;
                float most = 0.0f;
                if (row < rows) {
                    const T *src = static_cast<const T *>(a.q) + (long long)(s.first + row / a.group) * a.q_stride + (long long)(w.head * a.group + row % a.group) * D;
                    for (int d = lane; d < D; d += 32) most = fmaxf(most, fabsf(to_float(src[d])));
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (lane == 0) q_unit[r] = row_unit(most);
            }
            meet();
        }
        for (int i = tid; i < (C::ROWS / 16) * C::STEPS * 32; i += 32 * kWarps) {
            const int l = i & 31, ks = (i >> 5) % C::STEPS, mt = (i >> 5) / C::STEPS;
            const int d = ((l & 3) + 4 * (ks / (C::EC / 4))) * C::EC + 4 * (ks % (C::EC / 4));
            float x[2][4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int rr = mt * 16 + (l >> 2) + 8 * r, row = row0 + rr;
                const bool here = row < rows && d < D;
                const T *src = static_cast<const T *>(a.q) + (long long)(s.first + row / a.group) * a.q_stride + (long long)(w.head * a.group + row % a.group) * D + d;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[r][e] = here ? to_float(src[e]) : 0.0f;
                    if constexpr (HALF) x[r][e] *= q_unit[rr];
                }
            }
#pragma unroll
            for (int n = 0; n < C::NQ; ++n) {
                uint4 f;
                f.x = next_piece<HALF>(x[0][0], x[0][1], n == C::NQ - 1);
                f.y = next_piece<HALF>(x[1][0], x[1][1], n == C::NQ - 1);
                f.z = next_piece<HALF>(x[0][2], x[0][3], n == C::NQ - 1);
                f.w = next_piece<HALF>(x[1][2], x[1][3], n == C::NQ - 1);
                q_s[n * (C::ROWS / 16) * C::STEPS * 32 + i] = f;
            }
        }
        meet();
        const uint4 *q_w = q_s + (SPLITROWS ? warp * C::STEPS * 32 : 0) + lane;

        int limit[2];
        float factor[2];                             // of the scores, to the logarithm to base two
        const int wrow = row0 + (SPLITROWS ? warp * 16 : 0);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int rr = g + 8 * r;
            limit[r] = wrow + rr < rows ? limit_of(a, s, wrow + rr) : 0;
            factor[r] = a.cscale;
            if constexpr (HALF) factor[r] *= pow2_inverse(q_unit[wrow - row0 + rr]);
        }
        const int least_limit = wrow < rows ? limit_of(a, s, wrow) : 0;
        const int keys = tile_keys<C::ROWS>(a, s, w.tile);
        const int wlast = min(wrow + 16, rows) - 1;              // this warp's rows end here, and their keys
        const int wkeys = !SPLITROWS ? keys : wlast < wrow ? 0 : limit_of(a, s, wlast);

        float o[C::TILES][4], m[2], l[2];
        int unit = -126;                             // codes: o is divided by 2^unit, which follows the largest scale of the values
#pragma unroll
        for (int j = 0; j < C::TILES; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.0f;

        // ---- blocks of KB keys ------------------------------------------------------------------------------------
        constexpr int NG = C::KB / 16, NJ = C::KB / 8, BLOCKS = SPLITROWS ? C::UNIT / C::KB : 1;
        const int pitch = D * C::EB;
        for (int u = w.from; u < w.to; ++u, slot += 2) {
            const int ksl = slot % SLOTS, vsl = (slot + 1) % SLOTS;
            const uint8_t *k_at = ring + ksl * C::kSlotBytes, *v_at = ring + vsl * C::kSlotBytes;
            wait(&full[ksl], (slot / SLOTS) & 1, 11);
            const uint32_t there_all = *reinterpret_cast<volatile uint32_t *>(&there_s[ksl]);
            bool v_here = false;
#pragma unroll 1
            for (int blk = 0; blk < BLOCKS; ++blk) {
                const int k0 = (SPLITROWS ? blk : warp) * C::KB, p0 = u * C::UNIT + k0;      // the block's first key in its place, and in the sequence
                if (p0 >= wkeys) break;
                const uint32_t there = there_all >> (k0 / 16) & ((1u << NG) - 1);
                const bool partial = p0 + C::KB > wkeys || there != (1u << NG) - 1;          // places without keys
                const bool masked = p0 + C::KB > least_limit || there != (1u << NG) - 1;
                // scores: the main products, and apart from them those of the smaller pieces
                float z[NJ][4], zc[C::NQ > 1 ? NJ : 1][4];
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        z[j][e] = 0.0f;
                        if constexpr (C::NQ > 1) zc[j][e] = 0.0f;
                    }
                constexpr int PER = C::EC / 4;       // instructions a chunk
#pragma unroll
                for (int i = 0; i < C::NC; ++i) {
                    uint32_t kw[NJ][C::EC * C::EB / 4];
                    const int d = (t4 + 4 * i) * C::EC;
                    if constexpr (CUT) {
                    } else if (D == DP) {
#pragma unroll
                        for (int j = 0; j < NJ; ++j) read_words<C::EC * C::EB>(kw[j], k_at + (k0 + 8 * j + g) * (DP * C::EB) + d * C::EB);
                    } else {
#pragma unroll
                        for (int j = 0; j < NJ; ++j) {
#pragma unroll
                            for (int x = 0; x < C::EC * C::EB / 4; ++x) kw[j][x] = 0u;
                            if (d < D) read_words<C::EC * C::EB>(kw[j], k_at + (k0 + 8 * j + g) * pitch + d * C::EB);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < PER; ++x) {
                        uint4 q[C::NQ];
#pragma unroll
                        for (int n = 0; n < C::NQ; ++n) q[n] = q_w[n * (C::ROWS / 16) * C::STEPS * 32 + (i * PER + x) * 32];
#pragma unroll
                        for (int j = 0; j < NJ; ++j) {
                            uint32_t b[C::NK][2];
                            if constexpr (CUT) {
#pragma unroll
                                for (int n = 0; n < 3; ++n) read_words<8>(b[n], k_at + (((k0 / 8 + j) * C::NC + i) * 3 + n) * 256 + lane * 8);
                            } else if constexpr (C::CODED) {
                                codes_to_half<FMT>(kw[j][x], b[0][0], b[0][1]);
                            } else if constexpr (!C::F32) {
                                b[0][0] = kw[j][2 * x];
                                b[0][1] = kw[j][2 * x + 1];
                            } else {
                                float y[4] = {__uint_as_float(kw[j][0]), __uint_as_float(kw[j][1]), __uint_as_float(kw[j][2]), __uint_as_float(kw[j][3])};
#pragma unroll
                                for (int n = 0; n < 3; ++n) {
                                    b[n][0] = next_piece<false>(y[0], y[1], n == 2);
                                    b[n][1] = next_piece<false>(y[2], y[3], n == 2);
                                }
                            }
#pragma unroll
                            for (int order = C::NQ - 1; order >= 1; --order)
#pragma unroll
                                for (int n = 0; n <= order && n < C::NK; ++n) mma16<HALF>(zc[j], q[order - n], b[n][0], b[n][1]);
                            mma16<HALF>(z[j], q[0], b[0][0], b[0][1]);
                        }
                    }
                }
                float2 ks2[C::CODED ? NJ : 1], vs2[C::CODED ? NJ : 1];
                if constexpr (C::CODED)
#pragma unroll
                    for (int j = 0; j < NJ; ++j) ks2[j] = *reinterpret_cast<const float2 *>(k_at + C::UNIT * DP + (k0 + 8 * j + 2 * t4) * 4);
                if (!v_here) {
                    wait(&full[vsl], ((slot + 1) / SLOTS) & 1, 11);
                    v_here = true;
                }

                // ---- softmax ----------------------------------------------------------------------------------------------
                auto seen = [&](int j, int e) { return p0 + 8 * j + 2 * t4 + (e & 1) < limit[e >> 1] && (there >> (j >> 1) & 1); };
                float shrink = 1.0f;
                if constexpr (C::CODED) {
                    // P times the scales of the values, over 2^unit: at most 2^15
                    uint32_t most = 0;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        vs2[j] = *reinterpret_cast<const float2 *>(v_at + C::UNIT * DP + (k0 + 8 * j + 2 * t4) * 4);
                        if (partial) {
                            const int p = p0 + 8 * j + 2 * t4;
                            vs2[j].x = p < wkeys && (there >> (j >> 1) & 1) ? vs2[j].x : 0.0f;
                            vs2[j].y = p + 1 < wkeys && (there >> (j >> 1) & 1) ? vs2[j].y : 0.0f;
                        }
                        const uint32_t bx = __float_as_uint(vs2[j].x), by = __float_as_uint(vs2[j].y);
                        most = max(most, max(bx < 0x7F800000u ? bx : 0u, by < 0x7F800000u ? by : 0u));
                    }
                    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    const int e = max((int)(most >> 23) - 127 - 13, -126);       // (p <= 1, the scale < 2 * 2^13 then)
                    if (e > unit) {
                        shrink = ex2_approx((float)max(unit - e, -126));
                        unit = e;
                    }
                    const float down = __uint_as_float((uint32_t)(127 - min(unit, 126)) << 23);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        vs2[j].x *= down;
                        vs2[j].y *= down;
                    }
                }
                uint4 p[C::NQ][NG];
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = z[j][e];
                        if constexpr (C::NQ > 1) x += zc[j][e];
                        // (the two factors first: small queries and large keys, or the other way round, must not pass fp32's range on the way)
                        if constexpr (C::CODED) z[j][e] = x * (((e & 1) ? ks2[j].y : ks2[j].x) * factor[e >> 1]);
                        else z[j][e] = x * factor[e >> 1];
                    }
                if (masked) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) z[j][e] = seen(j, e) ? z[j][e] : -INFINITY;
                }
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], z[j][e]);
                float base[2], alpha[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                    const float now = fmaxf(m[r], top[r]);
                    base[r] = now == -INFINITY ? 0.0f : now;
                    alpha[r] = ex2_approx(m[r] - base[r]);
                    m[r] = now;
                    l[r] *= alpha[r];
                    alpha[r] *= shrink;
                }
                if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                    for (int j = 0; j < C::TILES; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[j][e] *= alpha[e >> 1];
                }
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y = ex2_approx(z[j][e] - base[e >> 1]);
                        l[e >> 1] += y;
                        z[j][e] = y;
                    }
                if constexpr (C::CODED) {
                    if (!masked) {
#pragma unroll
                        for (int j = 0; j < NJ; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) z[j][e] *= (e & 1) ? vs2[j].y : vs2[j].x;
                    } else {
                        // (the scale of a value that a row does not see may be anything)
#pragma unroll
                        for (int j = 0; j < NJ; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) z[j][e] = seen(j, e) ? z[j][e] * ((e & 1) ? vs2[j].y : vs2[j].x) : 0.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < NG; ++i)
#pragma unroll
                    for (int n = 0; n < C::NQ; ++n) {
                        p[n][i].x = next_piece<HALF>(z[2 * i][0], z[2 * i][1], n == C::NQ - 1);
                        p[n][i].y = next_piece<HALF>(z[2 * i][2], z[2 * i][3], n == C::NQ - 1);
                        p[n][i].z = next_piece<HALF>(z[2 * i + 1][0], z[2 * i + 1][1], n == C::NQ - 1);
                        p[n][i].w = next_piece<HALF>(z[2 * i + 1][2], z[2 * i + 1][3], n == C::NQ - 1);
                    }

                if (blk == BLOCKS - 1 || p0 + C::KB >= wkeys) leave(ksl);        // (what was read of it has been used: an arrival does not wait for loads)

                // ---- P V --------------------------------------------------------------------------------------------------
#pragma unroll
                for (int c = 0; c < C::NV; ++c) {
                    const int d = (g + 8 * c) * C::EV;
                    uint32_t vw[NG][4][C::EV * C::EB / 4];
                    if constexpr (CUT) {
                    } else if (D == DP && !partial) {
#pragma unroll
                        for (int x = 0; x < 4 * NG; ++x) read_words<C::EV * C::EB>(vw[x / 4][x % 4], v_at + (k0 + 8 * (x >> 1) + 2 * t4 + (x & 1)) * (DP * C::EB) + d * C::EB);
                    } else {
#pragma unroll
                        for (int x = 0; x < 4 * NG; ++x) {
                            const int in = 8 * (x >> 1) + 2 * t4 + (x & 1);
#pragma unroll
                            for (int y = 0; y < C::EV * C::EB / 4; ++y) vw[x / 4][x % 4][y] = 0u;
                            // (what lies in places without keys may be anything)
                            if (d < D && p0 + in < wkeys && (there >> (x / 4) & 1)) read_words<C::EV * C::EB>(vw[x / 4][x % 4], v_at + (k0 + in) * pitch + d * C::EB);
                        }
                    }
                    constexpr int W = C::CODED ? least_of(C::EV, 4) : 1;         // columns at a time: those of one word of codes
#pragma unroll
                    for (int e = 0; e < C::EV; e += W) {
                        uint32_t b[NG][W][C::NK][2];
#pragma unroll
                        for (int i = 0; i < NG; ++i) {
                            if constexpr (CUT) {
#pragma unroll
                                for (int n = 0; n < 3; ++n) read_words<8>(b[i][0][n], v_at + (((k0 / 16 + i) * C::TILES + c * C::EV + e) * 3 + n) * 256 + lane * 8);
                            } else {
#pragma unroll
                                for (int hf = 0; hf < 2; ++hf) {
                                    const uint32_t *w0 = vw[i][2 * hf], *w1 = vw[i][2 * hf + 1];
                                    if constexpr (C::CODED) {
                                        codes_to_half<FMT>(__byte_perm(w0[e / 4], w1[e / 4], 0x5140), b[i][0][0][hf], b[i][1][0][hf]);
                                        codes_to_half<FMT>(__byte_perm(w0[e / 4], w1[e / 4], 0x7362), b[i][2][0][hf], b[i][3][0][hf]);
                                    } else if constexpr (!C::F32) {
                                        b[i][0][0][hf] = __byte_perm(w0[e / 2], w1[e / 2], e & 1 ? 0x7632 : 0x5410);
                                    } else {
                                        float x = __uint_as_float(w0[e]), y = __uint_as_float(w1[e]);
#pragma unroll
                                        for (int n = 0; n < 3; ++n) b[i][0][n][hf] = next_piece<false>(x, y, n == 2);
                                    }
                                }
                            }
                        }
#pragma unroll
                        for (int x = 0; x < W; ++x) {
                            const int j = c * C::EV + e + x;
                            float d4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int order = C::NQ - 1; order >= 0; --order)
#pragma unroll
                                for (int n = 0; n <= order && n < C::NK; ++n)
#pragma unroll
                                    for (int i = 0; i < NG; ++i) mma16<HALF>(d4, p[order - n][i], b[i][x][n][0], b[i][x][n][1]);
#pragma unroll
                            for (int y = 0; y < 4; ++y) o[j][y] += d4[y];
                        }
                    }
                }
            }
            // (a warp without keys here gives the places back when they have come)
            if ((SPLITROWS ? 0 : warp * C::KB) + u * C::UNIT >= wkeys) leave(ksl);
            if (!v_here) wait(&full[vsl], ((slot + 1) / SLOTS) & 1, 11);
            leave(vsl);
        }
        const float grown = C::CODED ? __uint_as_float((uint32_t)(127 + min(unit, 126)) << 23) : 1.0f;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        if constexpr (C::CODED)
#pragma unroll
            for (int j = 0; j < C::TILES; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] *= grown;

        // ---- the tile's end ---------------------------------------------------------------------------------------
        const int part = run.part();
        if (part >= 0 && (part & 1)) cut = run.cut();
        float *dst = part < 0 ? nullptr : a.parts + (size_t)part * C::ROWS * (DP + 2);
        // columns of TILES' tile c * EV + e: values (2 t4 + 8 c) EV + e and (2 t4 + 1 + 8 c) EV + e
        if constexpr (!SPLITROWS) {
            // the warps' sums by way of shared memory: two of them leave theirs, the others add their own, then a warp joins four rows
            auto row_at = [&](int buf, int r) { return o_s + (buf * 16 + g + 8 * r) * C::kPad; };
            auto put = [&](int buf) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float *row = row_at(buf, r);
#pragma unroll
                    for (int c = 0; c < C::NV; ++c)
#pragma unroll
                        for (int e = 0; e < C::EV; ++e) {
                            row[(2 * t4 + 8 * c) * C::EV + e] = o[c * C::EV + e][2 * r];
                            row[(2 * t4 + 1 + 8 * c) * C::EV + e] = o[c * C::EV + e][2 * r + 1];
                        }
                    if (t4 == 0) ml_s[buf][g + 8 * r] = make_float2(m[r], l[r]);
                }
            };
            if (warp >= 2) put(warp - 2);
            meet();
            if (warp < 2) {
                float2 other[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) other[r] = ml_s[warp][g + 8 * r];
                __syncwarp();
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float now = fmaxf(m[r], other[r].x), base = now == -INFINITY ? 0.0f : now;
                    const float f0 = ex2_approx(m[r] - base), f1 = ex2_approx(other[r].x - base);
                    const float *row = row_at(warp, r);
                    m[r] = now;
                    l[r] = fmaf(l[r], f0, other[r].y * f1);
#pragma unroll
                    for (int c = 0; c < C::NV; ++c)
#pragma unroll
                        for (int e = 0; e < C::EV; ++e) {
                            float *x = &o[c * C::EV + e][2 * r];
                            x[0] = fmaf(x[0], f0, row[(2 * t4 + 8 * c) * C::EV + e] * f1);
                            x[1] = fmaf(x[1], f0, row[(2 * t4 + 1 + 8 * c) * C::EV + e] * f1);
                        }
                }
                put(warp);                           // (a thread reads and writes the same places)
            }
            meet();
            const bool store = !abort_flag;          // (behind the meeting: what a warp whose wait ran out has left there is in everybody's rows)
            for (int r = warp; r < 16; r += kWarps) {
                const int row = row0 + r;
                if (row >= rows) break;
                const float2 x0 = ml_s[0][r], x1 = ml_s[1][r];
                const float top = fmaxf(x0.x, x1.x), base = top == -INFINITY ? 0.0f : top;
                const float f0 = ex2_approx(x0.x - base), f1 = ex2_approx(x1.x - base), sum = fmaf(x0.y, f0, x1.y * f1);
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const long long t = s.first + row / a.group;
                T *out = static_cast<T *>(a.out) + t * a.out_stride + (long long)(w.head * a.group + row % a.group) * D;
                bool wild = false;
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) {
                    const int d = lane + 32 * i;
                    float y = fmaf(o_s[r * C::kPad + d], f0, o_s[(16 + r) * C::kPad + d] * f1);
                    if (dst) {
                        if (store) dst[(size_t)r * DP + d] = y;
                    } else {
                        y = sum == 0.0f ? 0.0f : y * inv;
                        wild = wild || (!finite(y) && sum == sum);
                        if (d < D && store) out[d] = from_float<T>(y);
                    }
                }
                if (dst) {
                    if (lane == 0 && store) reinterpret_cast<float2 *>(dst + C::ROWS * DP)[r] = make_float2(top, sum);
                } else if (__any_sync(0xffffffffu, wild) && lane == 0 && store) {
                    atomicOr(&mend_s, 1u << (number & 31));
                }
            }
        } else {
            const bool store = !abort_flag;
            bool wild = false;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int rr = warp * 16 + g + 8 * r, row = row0 + rr;
                const float sum = l[r], inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const bool here = row < rows && store;
                const long long t = s.first + row / a.group;
                T *out = static_cast<T *>(a.out) + t * a.out_stride + (long long)(w.head * a.group + row % a.group) * D;
#pragma unroll
                for (int c = 0; c < C::NV; ++c)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int e = 0; e < C::EV; ++e) {
                            const int d = (2 * t4 + x + 8 * c) * C::EV + e;
                            const float y = o[c * C::EV + e][2 * r + x];
                            if (dst) {
                                if (here) dst[(size_t)rr * DP + d] = y;
                            } else {
                                const float v = sum == 0.0f ? 0.0f : y * inv;
                                wild = wild || (here && !finite(v) && sum == sum);
                                if (here && d < D) out[d] = from_float<T>(v);
                            }
                        }
                if (dst && here && t4 == 0) reinterpret_cast<float2 *>(dst + C::ROWS * DP)[rr] = make_float2(m[r], sum);
            }
            if (__any_sync(0xffffffffu, wild) && lane == 0) atomicOr(&mend_s, 1u << (number & 31));
        }
    }
    meet();
    if (mend_s) mend_run<T, FMT, C::ROWS, C::UNIT, kThreads>(a, &start_s, mend_s, warp, kWarps, tops, meet);
    if (a.cuts && tid == 0) {
        a.cuts[blockIdx.x] = cut;
        a.whole[blockIdx.x] = !abort_flag;
    }
}

// ---- eight rows at most: single tokens -------------------------------------------------------------------------------------
// The products the other way round, S^T = K Q^T and O^T = V^T P^T: sixteen keys (or columns of V) by eight rows an instruction, so no half of it is empty, and half the registers hold the sums.  A thread
// takes its bytes of K and V as before; P^T as a result has its keys where the operand has its rows, and eight by eight of them are turned by one instruction.

template <typename T, int FMT, int DP>
struct TokenShape {
    using R = Shape<T, FMT, DP, false>;
    static constexpr bool F32 = R::F32, CODED = R::CODED, CUT = false;
    static constexpr int EB = R::EB, NQ = R::NQ, NK = R::NK, ROWS = 8, KB = R::KB, UNIT = kWarps * KB;
    static constexpr int EC = R::EC, NC = R::NC, EV = R::EV, NV = R::NV, STEPS = DP / 16, TILES = DP / 16;
    static constexpr int kQBytes = NQ * STEPS * 32 * 8, kPad = DP + 4, kOBytes = kWarps * 8 * kPad * 4;
    static constexpr int kSlotBytes = R::kSlotBytes;
    static constexpr int kBudget = (F32 && DP == 128 ? 112 : 74) * 1024;         // three blocks an SM (two where the sums of wide fp32 rows take the registers)
    static constexpr int kSlots = most_of(3, least_of(12, (kBudget - kQBytes - kOBytes - 1024) / kSlotBytes));
    static constexpr size_t kSmem = (size_t)kQBytes + kOBytes + (size_t)kSlots * kSlotBytes;
    static constexpr int kBlocks = kSmem > 112 * 1024 ? 1 : F32 && DP == 128 ? 2 : 3;
};

__device__ __forceinline__ uint32_t turned8(uint32_t x)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

template <typename T, int FMT, int DP>
__global__ void __launch_bounds__(kThreads, TokenShape<T, FMT, DP>::kBlocks)
paged_token_kernel(const __grid_constant__ AttnArgs a)
{
    using C = TokenShape<T, FMT, DP>;
    constexpr bool HALF = C::CODED;
    constexpr int SLOTS = C::kSlots;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;
    uint2 *q_s = reinterpret_cast<uint2 *>(smem + SLOTS * C::kSlotBytes);
    float *o_s = reinterpret_cast<float *>(smem + SLOTS * C::kSlotBytes + C::kQBytes);
    __shared__ uint64_t full[SLOTS], empty[SLOTS];
    __shared__ uint32_t there_s[SLOTS];
    __shared__ long long sums[kWarps + 3];
    __shared__ float2 ml_s[kWarps][8];
    __shared__ float q_unit[8];
    __shared__ volatile int abort_flag;
    __shared__ uint32_t mend_s;
    __shared__ typename Run<C::ROWS, C::UNIT, kThreads>::Start start_s;
    __shared__ int tops[kWarps];

    const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int D = a.c.D;
    if (tid == 0) {
        abort_flag = 0;
        mend_s = 0;
        for (int i = 0; i < SLOTS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kWarps);
        }
    }
    __syncthreads();
    dependency_wait();
    dependents_may_start();

    auto wait = [&](uint64_t *bar, uint32_t parity, int site) {
        const bool over = a.expire != 0 && expires_now(a.expire, site);
        if (!over && mbar_test(bar, parity)) return true;
        if (!abort_flag) {
            if (!over && mbar_wait(bar, parity)) return true;
            abort_flag = 1;
            atomicCAS(&g_rows_status, 0, site);
            linger();
        }
        return false;
    };
    Run<C::ROWS, C::UNIT, kThreads> run(a);
    bool more = run.begin(sums);
    if (more) run.keep(&start_s);
    if (warp == kWarps) {
        bring<C, kThreads>(a, run, more, ring, full, empty, there_s, wait);
        __syncwarp();
        if (abort_flag) linger();
        return;
    }

    auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); };
    auto leave = [&](int sl) {
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&empty[sl])) : "memory");
    };
    uint32_t slot = 0, number = 0;                   // of places; of the tile in the run
    int4 cut = make_int4(0, 0, 0, -1);
    for (; more; more = run.next(), ++number) {
        const Tile w = run.at();
        const Sequence &s = w.s;
        const int rows = (int)min((long long)s.n * a.group, 2147483647LL);
        const int row0 = w.tile * 8;

        // ---- Q as operands: a row's values by two warps' lanes, two rows a warp --------------------------------------------
        meet();                                      // (the tile before has been read)
        if constexpr (HALF) {
            for (int r = warp; r < 8; r += kWarps) {
                const int row = row0 + r;
                float most = 0.0f;
                if (row < rows) {
                    const T *src = static_cast<const T *>(a.q) + (long long)(s.first + row / a.group) * a.q_stride + (long long)(w.head * a.group + row % a.group) * D;
                    for (int d = lane; d < D; d += 32) most = fmaxf(most, fabsf(to_float(src[d])));
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (lane == 0) q_unit[r] = row_unit(most);
            }
            meet();
        }
        for (int i = tid; i < C::STEPS * 32; i += 32 * kWarps) {
            const int l = i & 31, ks = i >> 5, r = l >> 2, row = row0 + r;
            const int d = ((l & 3) + 4 * (ks / (C::EC / 4))) * C::EC + 4 * (ks % (C::EC / 4));
            const bool here = row < rows && d < D;
            const T *src = static_cast<const T *>(a.q) + (long long)(s.first + row / a.group) * a.q_stride + (long long)(w.head * a.group + row % a.group) * D + d;
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = here ? to_float(src[e]) : 0.0f;
                if constexpr (HALF) x[e] *= q_unit[r];
            }
#pragma unroll
            for (int n = 0; n < C::NQ; ++n) {
                uint2 f;
                f.x = next_piece<HALF>(x[0], x[1], n == C::NQ - 1);
                f.y = next_piece<HALF>(x[2], x[3], n == C::NQ - 1);
                q_s[n * C::STEPS * 32 + i] = f;
            }
        }
        meet();

        // this thread's rows: 2 t4 and 2 t4 + 1
        int limit[2];
        float factor[2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[C::TILES][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = row0 + 2 * t4 + r;
            limit[r] = row < rows ? limit_of(a, s, row) : 0;
            factor[r] = a.cscale;
            if constexpr (HALF) factor[r] *= pow2_inverse(q_unit[2 * t4 + r]);
        }
        const int least_limit = limit_of(a, s, row0), keys = tile_keys<8>(a, s, w.tile);
        int unit = -126;                             // codes: o is divided by 2^unit, which follows the largest scale of the values
#pragma unroll
        for (int j = 0; j < C::TILES; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
        // this thread's sums go to its places in shared memory, on top of what was put there before; `kept_m`: the reference maximum of that
        float kept_m[2] = {-INFINITY, -INFINITY};
        bool some = false;
        auto put = [&] {
            const float grown = C::CODED ? __uint_as_float((uint32_t)(127 + min(unit, 126)) << 23) : 1.0f;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float f = kept_m[r] == -INFINITY ? 0.0f : ex2_approx(kept_m[r] - m[r]);
                kept_m[r] = m[r];
                float *row = o_s + (warp * 8 + 2 * t4 + r) * C::kPad;
#pragma unroll
                for (int c = 0; c < C::NV; ++c)
#pragma unroll
                    for (int x = 0; x < C::EV / 2; ++x) {
                        const int j = c * (C::EV / 2) + x;
                        float2 *at = reinterpret_cast<float2 *>(row + (g + 8 * c) * C::EV + 2 * x);
                        float2 y = make_float2(o[j][r] * grown, o[j][2 + r] * grown);
                        if (some) y = make_float2(fmaf(at->x, f, y.x), fmaf(at->y, f, y.y));
                        *at = y;
                    }
            }
            some = true;
        };

        constexpr int NG = C::KB / 16;
        const int pitch = D * C::EB, k0 = warp * C::KB;
        for (int u = w.from; u < w.to; ++u, slot += 2) {
            if (!C::F32 && u > w.from && (u - w.from) % kKeptUnits == 0) {
                put();
#pragma unroll
                for (int j = 0; j < C::TILES; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
            }
            const int ksl = slot % SLOTS, vsl = (slot + 1) % SLOTS;
            const uint8_t *k_at = ring + ksl * C::kSlotBytes, *v_at = ring + vsl * C::kSlotBytes;
            const int p0 = u * C::UNIT + k0;         // the warp's first key in the sequence
            wait(&full[ksl], (slot / SLOTS) & 1, 11);
            if (p0 >= keys) {
                leave(ksl);
                wait(&full[vsl], ((slot + 1) / SLOTS) & 1, 11);
                leave(vsl);
                continue;
            }
            const uint32_t there = *reinterpret_cast<volatile uint32_t *>(&there_s[ksl]) >> (k0 / 16) & ((1u << NG) - 1);
            const bool partial = p0 + C::KB > keys || there != (1u << NG) - 1;
            const bool masked = p0 + C::KB > least_limit || there != (1u << NG) - 1;
            float z[NG][4], zc[C::NQ > 1 ? NG : 1][4];
#pragma unroll
            for (int i = 0; i < NG; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    z[i][e] = 0.0f;
                    if constexpr (C::NQ > 1) zc[i][e] = 0.0f;
                }
            constexpr int PER = C::EC / 4;           // instructions a chunk
#pragma unroll
            for (int i = 0; i < C::NC; ++i) {
                uint32_t kw[NG][2][C::EC * C::EB / 4];
                const int d = (t4 + 4 * i) * C::EC;
                if (D == DP) {
#pragma unroll
                    for (int j = 0; j < 2 * NG; ++j) read_words<C::EC * C::EB>(kw[j / 2][j % 2], k_at + (k0 + 8 * j + g) * (DP * C::EB) + d * C::EB);
                } else {
#pragma unroll
                    for (int j = 0; j < 2 * NG; ++j) {
#pragma unroll
                        for (int x = 0; x < C::EC * C::EB / 4; ++x) kw[j / 2][j % 2][x] = 0u;
                        if (d < D) read_words<C::EC * C::EB>(kw[j / 2][j % 2], k_at + (k0 + 8 * j + g) * pitch + d * C::EB);
                    }
                }
#pragma unroll
                for (int x = 0; x < PER; ++x) {
                    uint2 q[C::NQ];
#pragma unroll
                    for (int n = 0; n < C::NQ; ++n) q[n] = q_s[(n * C::STEPS + i * PER + x) * 32 + lane];
#pragma unroll
                    for (int j = 0; j < NG; ++j) {
                        uint4 f[C::NK];
                        if constexpr (C::CODED) {
                            codes_to_half<FMT>(kw[j][0][x], f[0].x, f[0].z);
                            codes_to_half<FMT>(kw[j][1][x], f[0].y, f[0].w);
                        } else if constexpr (!C::F32) {
                            f[0] = make_uint4(kw[j][0][2 * x], kw[j][1][2 * x], kw[j][0][2 * x + 1], kw[j][1][2 * x + 1]);
                        } else {
                            float y[2][4];
#pragma unroll
                            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                                for (int e = 0; e < 4; ++e) y[hf][e] = __uint_as_float(kw[j][hf][e]);
#pragma unroll
                            for (int n = 0; n < 3; ++n) {
                                f[n].x = next_piece<false>(y[0][0], y[0][1], n == 2);
                                f[n].y = next_piece<false>(y[1][0], y[1][1], n == 2);
                                f[n].z = next_piece<false>(y[0][2], y[0][3], n == 2);
                                f[n].w = next_piece<false>(y[1][2], y[1][3], n == 2);
                            }
                        }
#pragma unroll
                        for (int order = C::NQ - 1; order >= 1; --order)
#pragma unroll
                            for (int n = 0; n <= order && n < C::NK; ++n) mma16<HALF>(zc[j], f[n], q[order - n].x, q[order - n].y);
                        mma16<HALF>(z[j], f[0], q[0].x, q[0].y);
                    }
                }
            }
            float ks[C::CODED ? NG : 1][2], vs[C::CODED ? NG : 1][2];
            if constexpr (C::CODED)
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) ks[j][hf] = *reinterpret_cast<const float *>(k_at + C::UNIT * DP + (k0 + 16 * j + 8 * hf + g) * 4);
            wait(&full[vsl], ((slot + 1) / SLOTS) & 1, 11);

            // ---- softmax: element e of a tile is key g + 8 (e / 2) and row 2 t4 + e % 2 ---------------------------------
            float shrink = 1.0f;
            if constexpr (C::CODED) {
                uint32_t most = 0;
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const int in = 16 * j + 8 * hf + g;
                        float x = *reinterpret_cast<const float *>(v_at + C::UNIT * DP + (k0 + in) * 4);
                        if (partial && !(p0 + in < keys && (there >> j & 1))) x = 0.0f;
                        vs[j][hf] = x;
                        const uint32_t bits = __float_as_uint(x);
                        most = max(most, bits < 0x7F800000u ? bits : 0u);
                    }
                most = __reduce_max_sync(0xffffffffu, most);
                const int e = max((int)(most >> 23) - 127 - 13, -126);           // (p <= 1, the scale < 2 * 2^13 then)
                if (e > unit) {
                    shrink = ex2_approx((float)max(unit - e, -126));
                    unit = e;
                }
                const float down = __uint_as_float((uint32_t)(127 - min(unit, 126)) << 23);
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) vs[j][hf] *= down;
            }
            float top[2] = {-INFINITY, -INFINITY}, base[2], alpha[2];
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = z[j][e];
                    if constexpr (C::NQ > 1) x += zc[j][e];
                    // (the two factors first: small queries and large keys, or the other way round, must not pass fp32's range on the way)
                    if constexpr (C::CODED) z[j][e] = x * (ks[j][e >> 1] * factor[e & 1]);
                    else z[j][e] = x * factor[e & 1];
                }
            auto seen = [&](int j, int e) { return p0 + 16 * j + 8 * (e >> 1) + g < limit[e & 1] && (there >> j & 1); };
            if (masked) {
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[j][e] = seen(j, e) ? z[j][e] : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e & 1] = fmaxf(top[e & 1], z[j][e]);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], off));
                const float now = fmaxf(m[r], top[r]);
                base[r] = now == -INFINITY ? 0.0f : now;
                alpha[r] = ex2_approx(m[r] - base[r]);
                m[r] = now;
                l[r] *= alpha[r];
                alpha[r] *= shrink;
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                for (int j = 0; j < C::TILES; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][e] *= alpha[e & 1];
            }
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = ex2_approx(z[j][e] - base[e & 1]);
                    l[e & 1] += y;
                    z[j][e] = y;
                }
            if constexpr (C::CODED) {
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[j][e] *= vs[j][e >> 1];
                if (masked) {                        // (the scale of a value that a row does not see may be anything)
#pragma unroll
                    for (int j = 0; j < NG; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) z[j][e] = seen(j, e) ? z[j][e] : 0.0f;
                }
            }
            uint2 p[C::NQ][NG];
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int n = 0; n < C::NQ; ++n) {
                    p[n][j].x = turned8(next_piece<HALF>(z[j][0], z[j][1], n == C::NQ - 1));
                    p[n][j].y = turned8(next_piece<HALF>(z[j][2], z[j][3], n == C::NQ - 1));
                }
            leave(ksl);                              // (what was read of it has been used: an arrival does not wait for loads)

            // ---- O^T += V^T P^T: a tile is values 2 x and 2 x + 1 of each thread's chunk -----------------------------------
#pragma unroll
            for (int c = 0; c < C::NV; ++c) {
                const int d = (g + 8 * c) * C::EV;
                uint32_t vw[NG][4][C::EV * C::EB / 4];
                if (D == DP && !partial) {
#pragma unroll
                    for (int x = 0; x < 4 * NG; ++x) read_words<C::EV * C::EB>(vw[x / 4][x % 4], v_at + (k0 + 8 * (x >> 1) + 2 * t4 + (x & 1)) * (DP * C::EB) + d * C::EB);
                } else {
#pragma unroll
                    for (int x = 0; x < 4 * NG; ++x) {
                        const int in = 8 * (x >> 1) + 2 * t4 + (x & 1);
#pragma unroll
                        for (int y = 0; y < C::EV * C::EB / 4; ++y) vw[x / 4][x % 4][y] = 0u;
                        // (what lies in places without keys may be anything)
                        if (d < D && p0 + in < keys && (there >> (x / 4) & 1)) read_words<C::EV * C::EB>(vw[x / 4][x % 4], v_at + (k0 + in) * pitch + d * C::EB);
                    }
                }
#pragma unroll
                for (int x = 0; x < C::EV / 2; ++x) {
                    const int j = c * (C::EV / 2) + x;
                    float d4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    uint4 f[NG][C::NK];
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        if constexpr (C::CODED) {
                            const int word = x / 2, pick = x & 1 ? 0x7362 : 0x5140;
                            codes_to_half<FMT>(__byte_perm(vw[i][0][word], vw[i][1][word], pick), f[i][0].x, f[i][0].y);
                            codes_to_half<FMT>(__byte_perm(vw[i][2][word], vw[i][3][word], pick), f[i][0].z, f[i][0].w);
                        } else if constexpr (!C::F32) {
                            f[i][0] = make_uint4(__byte_perm(vw[i][0][x], vw[i][1][x], 0x5410), __byte_perm(vw[i][0][x], vw[i][1][x], 0x7632),
                                                 __byte_perm(vw[i][2][x], vw[i][3][x], 0x5410), __byte_perm(vw[i][2][x], vw[i][3][x], 0x7632));
                        } else {
                            float y[4][2];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
#pragma unroll
                                for (int e = 0; e < 2; ++e) y[k][e] = __uint_as_float(vw[i][k][2 * x + e]);
#pragma unroll
                            for (int n = 0; n < 3; ++n) {
                                f[i][n].x = next_piece<false>(y[0][0], y[1][0], n == 2);
                                f[i][n].y = next_piece<false>(y[0][1], y[1][1], n == 2);
                                f[i][n].z = next_piece<false>(y[2][0], y[3][0], n == 2);
                                f[i][n].w = next_piece<false>(y[2][1], y[3][1], n == 2);
                            }
                        }
                    }
                    if constexpr (C::F32) {
#pragma unroll
                        for (int order = C::NQ - 1; order >= 0; --order)
#pragma unroll
                            for (int n = 0; n <= order && n < C::NK; ++n)
#pragma unroll
                                for (int i = 0; i < NG; ++i) mma16<HALF>(d4, f[i][n], p[order - n][i].x, p[order - n][i].y);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[j][e] += d4[e];
                    } else {
#pragma unroll
                        for (int i = 0; i < NG; ++i) mma16<HALF>(o[j], f[i][0], p[0][i].x, p[0][i].y);
                    }
                }
            }
            leave(vsl);
        }

        // ---- the tile's end: the warps' sums by way of shared memory, two rows a warp --------------------------------------
        const int part = run.part();
        if (part >= 0 && (part & 1)) cut = run.cut();
        float *dst = part < 0 ? nullptr : a.parts + (size_t)part * 8 * (DP + 2);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], off);
            if (g == 0) ml_s[warp][2 * t4 + r] = make_float2(m[r], l[r]);
        }
        put();
        meet();
        const bool store = !abort_flag;              // (behind the meeting: what a warp whose wait ran out has left there is in everybody's rows)
        for (int r = warp; r < 8; r += kWarps) {
            const int row = row0 + r;
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
            T *out = static_cast<T *>(a.out) + t * a.out_stride + (long long)(w.head * a.group + row % a.group) * D;
            bool wild = false;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const int d = lane + 32 * i;
                float y = 0.0f;
#pragma unroll
                for (int x = 0; x < kWarps; ++x) y = fmaf(o_s[(x * 8 + r) * C::kPad + d], f[x], y);
                if (dst) {
                    if (store) dst[(size_t)r * DP + d] = y;
                } else {
                    y = sum == 0.0f ? 0.0f : y * inv;
                    wild = wild || (!finite(y) && sum == sum);
                    if (d < D && store) out[d] = from_float<T>(y);
                }
            }
            if (dst) {
                if (lane == 0 && store) reinterpret_cast<float2 *>(dst + 8 * DP)[r] = make_float2(top, sum);
            } else if (__any_sync(0xffffffffu, wild) && lane == 0 && store) {
                atomicOr(&mend_s, 1u << (number & 31));
            }
        }
    }
    meet();
    if (mend_s) mend_run<T, FMT, C::ROWS, C::UNIT, kThreads>(a, &start_s, mend_s, warp, kWarps, tops, meet);
    if (a.cuts && tid == 0) {
        a.cuts[blockIdx.x] = cut;
        a.whole[blockIdx.x] = !abort_flag;
    }
}

// The keys and values of UNIT positions of a sequence and head, fp32, as the three bf16 pieces of each, in the order of the operands of paged_rows_kernel's lanes (a place of its ring), so that they are cut
// once and not by each of its warps.  What lies behind the last key or in a page that is none becomes zeros; a sequence's first unit is always written.  Bound: memory (four bytes read, six written a value).
template <typename C>
__global__ void __launch_bounds__(128)
paged_cut_kernel(const PagedView c, uint8_t *k_out, uint8_t *v_out, int units)
{
    __shared__ long long rows_s[C::UNIT];
    dependency_wait();
    dependents_may_start();
    const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t4 = lane & 3, warp = tid >> 5, D = c.D;
    const int u = blockIdx.x % units, bh = blockIdx.x / units, b = bh / c.heads, head = bh % c.heads, p0 = u * C::UNIT;
    const Sequence s = sequence_of(c, b);
    if (s.n == 0 || (u > 0 && p0 >= s.len)) return;
    if (tid < C::UNIT) rows_s[tid] = p0 + tid < s.len ? row_of(c, b, head, p0 + tid) : -1;
    __syncthreads();
    auto read = [&](const uint8_t *from, int key, int d) {
        const long long at = rows_s[key];
        return at >= 0 && d < D ? __ldg(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(from) + at * D + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    };
    uint8_t *const k_to = k_out + (size_t)blockIdx.x * C::kSlotBytes + lane * 8, *const v_to = v_out + (size_t)blockIdx.x * C::kSlotBytes + lane * 8;
#pragma unroll 4
    for (int x = warp; x < C::UNIT / 8 * C::NC; x += 4) {
        const int j = x / C::NC, i = x % C::NC;
        float4 y = read(c.k, 8 * j + g, (t4 + 4 * i) * 4);
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            const uint32_t lo = next_piece<false>(y.x, y.y, n == 2), hi = next_piece<false>(y.z, y.w, n == 2);
            *reinterpret_cast<uint2 *>(k_to + (x * 3 + n) * 256) = make_uint2(lo, hi);
        }
    }
#pragma unroll 2
    for (int x = warp; x < C::UNIT / 16 * C::NV; x += 4) {
        const int i = x / C::NV, cc = x % C::NV;
        float y[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 f = read(c.v, 16 * i + 8 * (q >> 1) + 2 * t4 + (q & 1), (g + 8 * cc) * 4);
            y[q][0] = f.x; y[q][1] = f.y; y[q][2] = f.z; y[q][3] = f.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                const uint32_t lo = next_piece<false>(y[0][e], y[1][e], n == 2), hi = next_piece<false>(y[2][e], y[3][e], n == 2);
                *reinterpret_cast<uint2 *>(v_to + ((i * C::TILES + cc * 4 + e) * 3 + n) * 256) = make_uint2(lo, hi);
            }
    }
}

// fp32 keys and values are cut before the attention, into a buffer, where they serve several tiles of rows and that takes at most kMostCut bytes; without the memory, by the warps as ever.
// 16 heads over 8, before / by the warps, us: of 32, a sequence of 8192 keys, 64 rows 53 / 52, 128 57 / 59, 512 111 / 132, 2048 314 / 417, 32 sequences up to 512, 82 rows 65 / 63, 163 87 / 91, 327 127 / 149;
// of 64, 8192 keys, 128 rows 92 / 83, 256 123 / 135, 2048 572 / 849; of 128, 8192 keys, 32 rows 101 / 60, 64 114 / 117, 128 152 / 190, 2048 1336 / 2410.
constexpr size_t kMostCut = (size_t)1 << 30;
constexpr long long cut_rows(int width) { return width <= 32 ? 112 : width <= 64 ? 160 : 64; }
constexpr int kNoMemory = 1;                     // (no status code of the library)

template <typename T, int FMT, int DP, typename C>
int launch_kernel(void (*kern)(AttnArgs), AttnArgs a, cudaStream_t st)
{
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
    if (tiles < (1LL << 40) / most && tiles * most < grid) grid = (int)(tiles * most);
    const bool cuts = most > 1;
    StreamWorkspace::Lease ws;
    const size_t parts = cuts ? (size_t)2 * grid * C::ROWS * (DP + 2) * sizeof(float) : 0, lists = cuts ? ((size_t)grid * (sizeof(int4) + sizeof(int)) + 255) / 256 * 256 : 0;
    size_t pieces = 0;                           // bytes of K, and of V
    if constexpr (C::CUT) {
        const long long lots = (long long)a.c.B * a.c.heads;
        if (a.c.pages == 0 || a.c.most_pages == 0 || lots > (long long)(kMostCut / (2 * C::kSlotBytes)) / most) return kNoMemory;
        pieces = (size_t)lots * most * C::kSlotBytes;
    }
    if (cuts || pieces) {
        const int rc = g_paged_ws.enter(st, parts + lists + 2 * pieces, &ws);
        if (rc != HIPGPT_OK && pieces) {
            cudaGetLastError();
            return kNoMemory;
        }
        if (rc != HIPGPT_OK) return rc;
    }
    if (cuts) {
        a.parts = reinterpret_cast<float *>(ws.get());
        a.cuts = reinterpret_cast<int4 *>(ws.get() + parts);
        a.whole = reinterpret_cast<int *>(a.cuts + grid);
    }
    if constexpr (C::CUT) {
        a.cut_unit = C::UNIT;
        a.cut_k = ws.get() + parts + lists;
        a.cut_v = a.cut_k + pieces;
        a.cut_units = (int)most;
        e = launch_overlapped(paged_cut_kernel<C>, dim3((unsigned)(pieces / C::kSlotBytes)), dim3(128), 0, st, a.c, a.cut_k, a.cut_v, a.cut_units);
        if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "paged_cut_kernel: %s", cudaGetErrorString(e));
    }
    a.expire = take_expiry(1000);
    e = launch_overlapped(kern, dim3((unsigned)grid), dim3(kThreads), C::kSmem, st, a);
    if (e == cudaSuccess && cuts) e = launch_overlapped(paged_join_kernel<T, FMT, C::ROWS, DP>, dim3((unsigned)grid, (unsigned)(C::ROWS + 15) / 16), dim3(256), 0, st, a);
    return e == cudaSuccess ? check_launch("paged attention") : fail(HIPGPT_ERR_CUDA, "paged attention: %s", cudaGetErrorString(e));
}

// Rows a sequence, on the average: eight at most (single tokens of a small group), some, many.  32 sequences of up to 8192 keys, 8 heads, us with the three kernels (the third in bf16: tcgen05):
//   bf16 of 128     4 rows 114 / 118 / 171, 8 146 / 120 / 171, 15 229 / 168 / 173, 31 435 / 269 / 174;  e4m3 of 128  4 73 / 101 / 327, 8 94 / 104 / 328, 15 147 / 147 / 328, 31 265 / 233 / 330, 41 343 / 302 / 329
//   int8 of 64      4 53 / 63 / 305, 8 71 / 68 / 305, 31 198 / 146 / 305, 61 374 / 257 / 305
//   fp32 of 64      4 123 / 160 / 491, 8 161 / 161 / 491, 31 491 / 381 / 591, 61 936 / 694 / 943;  over int8 of 128  4 98 / 133 / 385, 8 126 / 134 / 385, 31 378 / 306 / 472, 61 715 / 558 / 762
// One limit for all types: plain bf16 of 17 to 32 rows and fp32 of 33 to 61 would be faster by the next kernel.
enum { kTokens, kSome, kMany };
template <typename T, int FMT, int DP>
int launch_width(int rows, const AttnArgs &a, cudaStream_t st)
{
    if (rows == kTokens) return launch_kernel<T, FMT, DP, TokenShape<T, FMT, DP>>(paged_token_kernel<T, FMT, DP>, a, st);
    if constexpr (sizeof(T) == 4 && FMT == HIPGPT_CACHE_PLAIN)
        if ((long long)a.c.T * a.group >= cut_rows(DP) * a.c.B) {
            const int rc = launch_kernel<T, FMT, DP, Shape<T, FMT, DP, true, true>>(paged_rows_kernel<T, FMT, DP, true, true>, a, st);
            if (rc != kNoMemory) return rc;
        }
    if constexpr (sizeof(T) == 4)
        if (rows == kMany) return launch_kernel<T, FMT, DP, Shape<T, FMT, DP, true>>(paged_rows_kernel<T, FMT, DP, true>, a, st);
    return launch_kernel<T, FMT, DP, Shape<T, FMT, DP, false>>(paged_rows_kernel<T, FMT, DP, false>, a, st);
}
template <typename T, int FMT>
int launch_format(int rows, const AttnArgs &a, cudaStream_t st)
{
    return a.c.D <= 32 ? launch_width<T, FMT, 32>(rows, a, st) : a.c.D <= 64 ? launch_width<T, FMT, 64>(rows, a, st) : launch_width<T, FMT, 128>(rows, a, st);
}

template <typename T>
int launch_paged(int format, const AttnArgs &a, cudaStream_t st)
{
    const long long all = (long long)a.c.T * a.group;
    const int rows = all <= 8LL * a.c.B ? kTokens : all <= 32LL * a.c.B ? kSome : kMany;
    if (sizeof(T) == 2 && rows == kMany && a.c.pages > 0) return launch_paged_tc(format, a, st);         // (without pages there is nothing to copy)
    return format == HIPGPT_CACHE_PLAIN ? launch_format<T, HIPGPT_CACHE_PLAIN>(rows, a, st)
         : format == HIPGPT_CACHE_E4M3  ? launch_format<T, HIPGPT_CACHE_E4M3>(rows, a, st) : launch_format<T, HIPGPT_CACHE_INT8>(rows, a, st);
}

}  // namespace

void paged_release_scratch() { g_paged_ws.release(); }

int paged_rows_status_fetch(int *status)
{
    int s = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&s, g_rows_status, sizeof(int));
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "cudaMemcpyFromSymbol: %s", cudaGetErrorString(e));
    if (s != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_rows_status, &zero, sizeof(int));
    }
    *status = s;
    return HIPGPT_OK;
}

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
    a.cscale = scale * kLog2e;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return cache->type == HIPGPT_TYPE_F32 ? launch_paged<float>(cache->format, a, st) : launch_paged<__nv_bfloat16>(cache->format, a, st);
}
