// Attention of new tokens over a paged cache on the tensor pipe (tcgen05 + TMEM): 16-bit activations with many rows a sequence, every cache format.
//
// A block takes 256 rows (two tiles of 128, a row a TMEM lane) of one sequence and head of the cache, so the keys and values that it fetches serve both; one block an SM, which
// goes from one run of units of 128 keys to the next (attn_paged.cuh).  Roles:
//   warps 0-3, 4-7   softmax of the first and of the second tile, a thread a row: its scores are read from TMEM into registers, P = exp2(s - m) goes over them in
//                    bf16.  The reference maximum m moves, and the sums so far are scaled, when a row of the warp has outgrown it by more than 2^8 (P in bf16 and
//                    sums in fp32 do not care).  P V is summed in TMEM.
//   warps 8-11       codes that were not widened before the kernel: widen them to fp16 in the layout of the operands, two tiles of keys and of values ahead, times their scales over a power of two of each 64 keys, which goes
//                    into the scores' factor, and for V into the exponent of P.  (e4m3: exact; int8: values are rounded to fp16, as P is, scores multiplied by the keys' scales instead.)
//                    Plain and widened rows: one warp clears the rows of V behind the last key, which may hold anything.
//   warp 12          (codes widened here: and 14, one for each tile) issues the products: P V of a tile, 64 keys as soon as the softmax has them, then Q K^T of its next keys over the same columns of TMEM (products of one thread run in
//                    the order of their issue, so a commit behind the second covers the first); the other tile's softmax runs meanwhile.
//   warp 13          asks for the copies, a lane a run of keys in one page: boxes of 64 columns, swizzled, straight into the operands (plain; a page that is none lies
//                    outside the tensor and comes as zeros), or codes and scales as they lie into a ring of half tiles.  (Loads by the threads themselves, 16 KB on their way, brought
//                    6 bytes a clock; bulk copies bring 24.)
// Bound: neither pipe yet.  At D = 128 a unit's products are 2048 clocks of the tensor pipe and its exponentials as many of the special-function unit; plain rows take 4150, the chain from P to the next scores
// (P V's second half, Q K^T, two commits: 1750) and the softmax (2300) of a tile one after the other, the two tiles half a turn apart.  Widening codes here takes 6500 (four half
// tiles of 1600).  32 heads over 8 of 128: five ragged sequences of 1100 new tokens in 8000, plain: 423 us, 903 TFLOP/s; 4096 new tokens in 32768, int8: 2.18 ms, 946 TFLOP/s, widened before;
// 3.10 ms, widened here.
// Every wait is bounded: on expiry the block raises a flag that cuts all later waits short, records a status code, skips its stores, lets what is on its way land,
// frees its TMEM and returns.
#include "attn_paged.cuh"
#include "stream_workspace.hpp"
#include "tma_host.cuh"

#include <math.h>

namespace hipgpt {

extern StreamWorkspace g_paged_ws;

namespace {

constexpr int kRows = 256, kKeys = 128, kStages = 2;
constexpr int kTables = 4;            // a tile's scales and pages are read until its scores have been: the products of the tile after the next say so
constexpr int kWideners = 128, kThreads = 512;
// Registers a thread of each warpgroup: 128 at launch; 184 + 184 + 88 + 56 = 4 x 128, and where no codes are widened here 200 + 200 + 56 + 56 (4096 tokens over 32768 int8 keys: 2205 -> 2148 us)
template <bool WIDENS> constexpr int kSoftRegs = WIDENS ? 184 : 200;
template <bool WIDENS> constexpr int kWidenRegs = WIDENS ? 88 : 56;
constexpr int kIssueRegs = 56;
constexpr int kHalf = 64, kSlots = 3;  // keys of a half tile of codes, half tiles in the ring
constexpr float kRescaleStep = 8.0f;
// Units after which the sums in TMEM are added to what the block keeps of them in memory: the tensor pipe cuts off towards zero, 2^-24 to 2^-23 of the sum for each sixteen keys, so after 32768 keys 2^-12 at most, an
// eighth of what rounding a result to bf16 may take.  (Every 64 units: 9 % of a long call.)
constexpr int kKept = 256;
constexpr uint32_t kTmemCols = 512, kColS = 0, kColO = 256;

__device__ int g_paged_status = 0;

// (in line: with calls inside them the roles' registers cannot be shared out)
__device__ __forceinline__ bool wait_slow(uint64_t *bar, uint32_t parity, int site, volatile int *abort_flag)
{
    if (mbar_wait(bar, parity)) return true;
    *abort_flag = 1;
    atomicCAS(&g_paged_status, 0, site);
    linger();
    return false;
}

// The largest scale of 64 keys goes to [2^k, 2^(k + 1)) in fp16: 128 * 2^8 and 448 * 2^7 are still numbers there, and rows whose scale is 2^-21 of it keep their digits
template <int FMT> constexpr int kUp = FMT == HIPGPT_CACHE_E4M3 ? 6 : 7;
// ... and values whose own power of two is 2^-kFar of those before them take 2^-kFar of that: they need not fill fp16, and the exponents that P takes from tile to tile stay near each other
constexpr int kFar = 20;

// Codes that were widened before the call's attention: rows of fp16 of each sequence and head, one behind the other
struct Wide {
    void *k, *v;                         // [sequence][head][room][D]
    float *scale;                        // [sequence][head][room]: int8, the scales of the keys over their 64's power of two
    float *k_unit, *v_exp;               // [sequence][head][room / 64]
    int room;                            // keys, a multiple of 128
};

template <int FMT, int DP, bool WIDENED>
struct TcCfg {
    static constexpr int kQTile = 128 * DP * 2, kTile = kKeys * DP * 2, kSlot = kHalf * DP;
    static constexpr size_t kBytes = 2 * (size_t)kQTile + 2 * kStages * (size_t)kTile + (FMT == HIPGPT_CACHE_PLAIN || WIDENED ? 0 : kSlots * (size_t)kSlot) + 1024;
};

template <int FMT, int DP, bool WIDENED>
__global__ void __launch_bounds__(kThreads, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttnArgs a, const Wide wide, int expire)
{
    using C = TcCfg<FMT, DP, WIDENED>;
    using T = __nv_bfloat16;
    constexpr bool CODED = FMT != HIPGPT_CACHE_PLAIN, SCALED = FMT == HIPGPT_CACHE_INT8, WIDENS = CODED && !WIDENED;
    constexpr float kBias = CODED ? 6.0f : 0.0f;
    constexpr int kIssuers = WIDENS ? 2 : 1;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *q_s = base;                             // [tile][block of 64 columns][128 rows][128 B], swizzled
    uint8_t *k_s = q_s + 2 * C::kQTile;              // [stage][block][128 keys][128 B], K-major operand
    uint8_t *v_s = k_s + kStages * C::kTile;         // the same bytes, read as an N-major operand
    uint8_t *raw_s = v_s + kStages * C::kTile;       // [slot][64 keys][D] codes as they lie in their pages
    __shared__ uint64_t k_full[kStages], v_full[kStages], k_free[kStages], v_free[kStages], q_full[2], s_full[2], p_full[2][2], o_done[2];
    __shared__ uint64_t landed[WIDENS ? kSlots : kStages], raw_free[kSlots];
    __shared__ __align__(16) float scale_s[WIDENS ? kSlots : 1][kHalf];
    __shared__ __align__(16) float ks_s[SCALED ? kTables : 1][kKeys];       // int8: the scales of the keys, over their 64's power of two
    __shared__ float k_unit[kTables][2], v_exp[kTables][2];          // codes: the power of two that each 64 keys of a tile were divided by, the exponent of that of the values
    __shared__ float q_unit[CODED ? 2 * 128 : 1];                    // and that of a row of Q
    __shared__ uint32_t there_s[kTables];            // whether each 16 keys of a tile have a page
    __shared__ long long sums[kThreads / 32 + 2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    __shared__ uint32_t mend_s;                      // tiles of the run (their numbers modulo 32) with rows to look at again
    __shared__ typename Run<kRows, kKeys, kThreads>::Start start_s;
    __shared__ int tops[8];

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (tid == 0) {
        abort_flag = 0;
        mend_s = 0;
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&k_full[i], WIDENS ? kWideners / 32 : 1);
            mbar_init(&v_full[i], WIDENS ? kWideners / 32 : 1);
            mbar_init(&k_free[i], kIssuers);
            mbar_init(&v_free[i], kIssuers);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 4);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i][0], 4);
            mbar_init(&p_full[i][1], 4);
            mbar_init(&o_done[i], 1);
        }
        for (int i = 0; i < (WIDENS ? kSlots : kStages); ++i) mbar_init(&landed[i], 1);
        for (int i = 0; i < kSlots; ++i) mbar_init(&raw_free[i], kWideners / 32);
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = 0;                         // all 512 columns are this block's
    dependency_wait();
    dependents_may_start();

    // site codes in the status word: 1 keys landed, 2 values landed, 3 queries there, 4 scores ready, 5 probabilities written, 6 sums complete, 7 key stage free, 8 value stage free, 9 copies landed,
    // 10 half tile free
    // (what has come costs one test and no look at the flag: there are seven waits for each 128 keys in the warp that issues the products)
    bool seen = true;                                // what this thread waited for last has come (for who asks for copies then)
    auto wait = [&](uint64_t *bar, uint32_t parity, int site) {
        seen = true;
        if (expire != 0 && expires_now(expire, site) && !abort_flag) {
            abort_flag = 1;
            atomicCAS(&g_paged_status, 0, site);
            linger();
            seen = false;
        } else if (!mbar_test(bar, parity)) {
            seen = !abort_flag && wait_slow(bar, parity, site, &abort_flag);
        }
    };
    auto arrive = [&](uint64_t *bar) {
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
    };

    Run<kRows, kKeys, kThreads> run(a);
    bool more = run.begin(sums);
    if (more) run.keep(&start_s);
    // units of each of the two tiles of rows within the block's run of the tile: [from, to) cut to what the tile's rows see (the second has no rows where there are none)
    auto units_of = [&](const Tile &w, int half) {
        const long long rows = (long long)w.s.n * a.group, first = (long long)w.tile * kRows + 128 * half;
        if (first >= rows) return 0;
        const long long last = min(first + 128, rows) - 1;
        const int u = max(1, (limit_of(a, w.s, (int)last) + kKeys - 1) / kKeys);
        return max(min(w.to, u) - w.from, 0);
    };

    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        more = more && (warp < 14 || (warp == 14 && kIssuers == 2));             // (registers are given back by whole warpgroups)
    }
    if (warp == 13 || warp == 15) {
        // ================= the copies ============================================================================
        uint32_t n = 0, slot = 0;                    // tiles of keys so far; half tiles of codes
        const int page_keys = 1 << a.c.shift, D = a.c.D;
        for (; more; more = run.next()) {
            const Tile w = run.at();
            const int units = max(units_of(w, 0), units_of(w, 1)), keys = tile_keys<kRows>(a, w.s, w.tile);
            // the pages of a tile's eight times sixteen keys, a lane each; asked for a tile ahead
            auto look = [&](int u) {
                const int p = u * kKeys + 16 * lane;
                const int pg = lane < 8 && p < keys ? __ldg(a.c.table + (size_t)w.b * a.c.most_pages + (p >> a.c.shift)) : -1;
                return pg < a.c.pages ? pg : -1;
            };
            int page = look(w.from);
            for (int u = w.from; u < w.from + units; ++u, ++n) {
                const int st = n % kStages, p0 = u * kKeys;
                const uint32_t ph = (n / kStages) & 1;
                const uint32_t there = __ballot_sync(0xffffffffu, page >= 0) & 255u;
                const int next_page = u + 1 < w.from + units ? look(u + 1) : -1;
                if (lane == 0) there_s[n % kTables] = there;         // (before the arrivals below)
                if constexpr (!WIDENS) {
                    constexpr int NB = DP / 64;
                    const int run_keys = WIDENED ? kKeys : min(page_keys, kKeys), runs = kKeys / run_keys;
                    const int at = lane / NB * run_keys, x = lane % NB * 64;                    // this lane's box
                    const int pg = __shfl_sync(0xffffffffu, page, (at >> 4) & 7);
                    const int z = WIDENED ? w.b * a.c.heads + w.head : pg < 0 ? a.c.pages * a.c.heads : pg * a.c.heads + w.head;
                    const int y = WIDENED ? p0 : (p0 + at) & (page_keys - 1);
#pragma unroll
                    for (int which = 0; which < 2; ++which) {
                        if (n >= kStages) wait(which ? &v_free[st] : &k_free[st], ph ^ 1, which ? 8 : 7);
                        uint64_t *bar = which ? &landed[st] : &k_full[st];
                        __syncwarp();
                        if (lane == 0 && seen) mbar_arrive_expect_tx(bar, (uint32_t)C::kTile);
                        __syncwarp();
                        if (lane < runs * NB && seen)
                            tma_load_3d((which ? v_s : k_s) + st * C::kTile + (x / 64) * (kKeys * 128) + at * 128, which ? &vmap : &kmap, x, y, z, bar);
                    }
                } else {
                    const int run_keys = min(page_keys, kHalf), runs = kHalf / run_keys;
#pragma unroll
                    for (int part = 0; part < 4; ++part, slot = slot + 1) {
                        const int which = part >> 1, sl = slot % kSlots, at = (part & 1) * kHalf + lane * run_keys;
                        const int pg = __shfl_sync(0xffffffffu, page, (at >> 4) & 7);
                        const int count = lane < runs && pg >= 0 ? min(run_keys, keys - (p0 + at)) : 0;             // (a page that is none lies behind the last key)
                        const int scales = (count + 3) & ~3;         // whole 16 bytes, within the page
                        int bytes = count * D + scales * 4;
#pragma unroll
                        for (int o = 1; o < 4; o <<= 1) bytes += __shfl_xor_sync(0xffffffffu, bytes, o);             // (runs are four at most)
                        if (slot >= kSlots) wait(&raw_free[sl], ((slot / kSlots) & 1) ^ 1, 10);
                        __syncwarp();
                        if (lane == 0 && seen) mbar_arrive_expect_tx(&landed[sl], (uint32_t)bytes);
                        __syncwarp();
                        if (count > 0 && seen) {
                            const long long row = ((((long long)pg * a.c.heads) + w.head) << a.c.shift) + ((p0 + at) & (page_keys - 1));
                            bulk_load(raw_s + sl * C::kSlot + lane * run_keys * D, (which ? a.c.v : a.c.k) + row * D, (uint32_t)(count * D), &landed[sl]);
                            bulk_load(&scale_s[sl][lane * run_keys], (which ? a.c.vs : a.c.ks) + row, (uint32_t)(scales * 4), &landed[sl]);
                        }
                    }
                }
                page = next_page;
            }
        }
        __syncwarp();
        if (abort_flag) linger();
    } else if (warp >= 8 && warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWidenRegs<WIDENS>));
        // ================= codes to operands; rows behind the last key ===========================================
        const int pt = tid - 256, D = a.c.D;
        uint32_t n = 0, slot = 0;
        int v_most = 0;                              // the largest exponent of values so far
        if constexpr (!WIDENS) more = more && warp == 8;
        for (; more; more = run.next()) {
            const Tile w = run.at();
            const int units = max(units_of(w, 0), units_of(w, 1)), keys = tile_keys<kRows>(a, w.s, w.tile);
            v_most = -200;
            // (widened: the scales of a tile's keys, and the two powers of two of its keys and of its values, a tile ahead)
            float4 scales = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float unit = 0.0f;
            auto fetch = [&](int u) {
                const size_t bh = (size_t)w.b * a.c.heads + w.head;
                if constexpr (SCALED) scales = *reinterpret_cast<const float4 *>(wide.scale + bh * wide.room + u * kKeys + lane * 4);
                if (lane < 4) unit = (lane < 2 ? wide.k_unit : wide.v_exp)[bh * (wide.room / kHalf) + u * 2 + (lane & 1)];
            };
            if constexpr (WIDENED) if (units > 0) fetch(w.from);
            for (int u = w.from; u < w.from + units; ++u, ++n) {
                const int st = n % kStages, p0 = u * kKeys;
                const uint32_t ph = (n / kStages) & 1;
                if constexpr (!WIDENS) {
                    wait(&landed[st], ph, 9);
                    if constexpr (WIDENED) {
                        if constexpr (SCALED) *reinterpret_cast<float4 *>(&ks_s[n % kTables][lane * 4]) = scales;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int e = (int)__shfl_sync(0xffffffffu, unit, 2 + h), x = max(e, v_most - kFar), d = x - e;
                            v_most = max(v_most, x);
                            if (lane == 2 + h) unit = (float)x;
                            if (d > 0) {             // (seldom: the kernel before did not know those before)
                                const uint32_t f = d < 15 ? (uint32_t)(15 - d) << 10 : d < 25 ? 1u << (24 - d) : 0u, f2 = f | f << 16;
                                for (int i = lane; i < kHalf * 8; i += 32)
#pragma unroll
                                    for (int nb = 0; nb < DP / 64; ++nb) {
                                        uint4 *at = reinterpret_cast<uint4 *>(v_s + st * C::kTile + nb * (kKeys * 128) + h * (kHalf * 128) + i * 16);
                                        const uint4 w = *at;
                                        *at = make_uint4(mul_f16x2(w.x, f2), mul_f16x2(w.y, f2), mul_f16x2(w.z, f2), mul_f16x2(w.w, f2));
                                    }
                                proxy_fence();
                            }
                        }
                        if (lane < 4) (lane < 2 ? k_unit : v_exp)[n % kTables][lane & 1] = unit;
                        if (u + 1 < w.from + units) fetch(u + 1);
                    }
                    const int first = keys - p0;
                    if (first < kKeys) {
                        for (int i = max(first, 0) * 8 + lane; i < kKeys * 8; i += 32)
#pragma unroll
                            for (int nb = 0; nb < DP / 64; ++nb) *reinterpret_cast<uint4 *>(v_s + st * C::kTile + nb * (kKeys * 128) + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                        proxy_fence();
                    }
                    arrive(&v_full[st]);
                } else {
                    constexpr int CH = DP / 16, PER = kWideners / CH, N = kHalf / PER;       // chunks of 16 codes a key; keys at a time; rounds
                    const int c = pt % CH, k0 = pt / CH;
                    // the two halves of a chunk's 32 bytes; where two threads of a row would meet in a bank, one takes them the other way round
                    const int c0 = 2 * c, turn = DP == 128 ? c >> 2 : 0;
                    uint32_t there = 0;
                    bool all = false;
#pragma unroll 1
                    for (int part = 0; part < 4; ++part, ++slot) {
                        const int which = part >> 1, sl = slot % kSlots, base_key = (part & 1) * kHalf;
                        wait(&landed[sl], (slot / kSlots) & 1, 9);
                        if (part == 0) {
                            there = *reinterpret_cast<volatile uint32_t *>(&there_s[n % kTables]);
                            all = p0 + kKeys <= keys && there == 255u && D == DP;
                        }
                        auto holds = [&](int key) { return all || (p0 + base_key + key < keys && (there >> ((base_key + key) >> 4) & 1)); };
                        uint4 raw[N];
                        float scale[N];
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            const int key = k0 + PER * i;
                            const bool ok = holds(key) && c * 16 < D;
                            raw[i] = ok ? *reinterpret_cast<const uint4 *>(raw_s + sl * C::kSlot + key * D + c * 16) : make_uint4(0u, 0u, 0u, 0u);
                            scale[i] = ok ? scale_s[sl][key] : 0.0f;
                        }
                        uint32_t most = 0;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t bits = holds(lane + 32 * i) ? __float_as_uint(scale_s[sl][lane + 32 * i]) : 0u;
                            most = max(most, bits < 0x7F800000u ? bits : 0u);
                        }
                        most = __reduce_max_sync(0xffffffffu, most);
                        int e = (int)(most >> 23) - 127 - kUp<FMT>;
                        if (which) {
                            // Values far below those before them need not fill fp16, and all of one size with P: a tile of zeros must not carry the sum of exponentials out of fp32
                            e = max(max(e, v_most - kFar), -96);
                            v_most = max(v_most, e);
                        }
                        e = min(max(e, -126), 120);
                        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                        float key_scale = 0.0f;
                        if (SCALED && !which && pt < kHalf) key_scale = holds(pt) ? scale_s[sl][pt] * down : 0.0f;
                        if (n >= kStages && (part & 1) == 0) wait(which ? &v_free[st] : &k_free[st], ph ^ 1, which ? 8 : 7);
                        if (pt == 0) {
                            if (which) v_exp[n % kTables][part & 1] = (float)e;
                            else k_unit[n % kTables][part & 1] = __uint_as_float((uint32_t)(127 + e) << 23);
                        }
                        if constexpr (SCALED)
                            if (which == 0 && pt < kHalf) ks_s[n % kTables][base_key + pt] = key_scale;
                        uint8_t *tile = (which ? v_s : k_s) + st * C::kTile + (c0 / 8) * (kKeys * 128) + base_key * 128;
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            const uint32_t in[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w}, s2 = SCALED && !which ? 0x3C003C00u : half2_of(scale[i] * down, scale[i] * down);
                            uint32_t out[8];
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                codes_to_half<FMT>(in[x], out[2 * x], out[2 * x + 1]);
                                out[2 * x] = mul_f16x2(out[2 * x], s2);
                                out[2 * x + 1] = mul_f16x2(out[2 * x + 1], s2);
                            }
                            const int key = k0 + PER * i;
                            const uint4 lo = make_uint4(out[0], out[1], out[2], out[3]), hi = make_uint4(out[4], out[5], out[6], out[7]);
                            *reinterpret_cast<uint4 *>(tile + sw128(key, (c0 + turn) % 8)) = turn ? hi : lo;
                            *reinterpret_cast<uint4 *>(tile + sw128(key, (c0 + 1 - turn) % 8)) = turn ? lo : hi;
                        }
                        arrive(&raw_free[sl]);       // (not before the codes have been used: an arrival does not wait for loads)
                        if (part & 1) {
                            proxy_fence();
                            arrive(which ? &v_full[st] : &k_full[st]);
                        }
                    }
                }
            }
        }
    } else if (warp >= 12) {
        // ================= the products =========================================================================
        // Plain and widened rows: one warp issues those of both tiles, one tile's after the other's, so that one tile's softmax runs beside the other's products.  (Two warps' products share the pipe, and
        // both tiles' scores come late, at the same time: 442 against 422 us.)  Codes: a warp for each tile, because they wait for the values to be widened and must not wait for each other too.
        constexpr uint32_t kHalfTypes = CODED ? ~((1u << 7) | (1u << 10)) : ~0u;         // fp16 operands instead of bf16
        constexpr uint32_t idesc_qk = idesc_bf16(128, kKeys, 0) & kHalfTypes, idesc_pv = idesc_bf16(128, DP, 1) & kHalfTypes;
        const int h0 = kIssuers == 2 ? (warp - 12) >> 1 : 0, h1 = kIssuers == 2 ? h0 + 1 : 2;      // the tiles of this warp
        uint32_t n = 0, np[2] = {0, 0}, items = 0;   // tiles of keys, of probabilities; tiles of rows
        for (; more; more = run.next(), ++items) {
            const Tile w = run.at();
            // (read from one lane: every address below is then known to be the warp's, not a lane's)
            const int u[2] = {__shfl_sync(0xffffffffu, units_of(w, 0), 0), __shfl_sync(0xffffffffu, units_of(w, 1), 0)}, units = max(u[0], u[1]);
            const int mine = kIssuers == 2 ? u[h0] : units;
            auto ph = [&](int t) { return ((n + t) / kStages) & 1u; };
            // the last of this warp's to read a stage gives it back
            auto last = [&](int half, int t) { return kIssuers == 2 || half == (t < u[1] ? 1 : 0); };
            auto qk = [&](int half, int t) {
                const int st = (n + t) % kStages;
                const uint64_t dq = make_desc(smem_u32(q_s + half * C::kQTile), 16, 1024, 2), dk = make_desc(smem_u32(k_s + st * C::kTile), 16, 1024, 2);
                if (kIssuers == 2 || half == (t < u[0] ? 0 : 1)) {           // (the first to need it)
                    wait(&k_full[st], ph(t), 1);
                    tc_fence_after();
                }
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        const uint64_t off = (uint64_t)((k / 4) * (128 * 128 / 16) + (k % 4) * 2);
                        mma_h_ss(tmem + kColS + half * 128, dq + off, dk + off, idesc_qk, k ? 1u : 0u);
                    }
                    tc_commit(&s_full[half]);
                    if (last(half, t)) tc_commit(&k_free[st]);
                }
            };
            for (int half = h0; half < h1; ++half) wait(&q_full[half], items & 1, 3);       // (without units too: a phase must not be passed over)
            tc_fence_after();
            for (int half = h0; half < h1; ++half) {
                if (u[half]) qk(half, 0);
                else if (elect_one()) tc_commit(&o_done[half]);      // (whoever has no units of this tile must not run ahead into the next)
            }
            for (int t = 0; t < mine; ++t) {
                const int st = (n + t) % kStages;
                const uint64_t dv = make_desc(smem_u32(v_s + st * C::kTile), kKeys * 128, 1024, 2);
                wait(&v_full[st], ph(t), 2);
                for (int half = h0; half < h1; ++half) {
                    if (t >= u[half]) continue;
#pragma unroll
                    for (int part = 0; part < 2; ++part) {               // (the first 64 keys while the softmax takes the others)
                        wait(&p_full[half][part], np[half] & 1, 5);
                        tc_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (int k = part * (kKeys / 32); k < (part + 1) * (kKeys / 32); ++k)
                                mma_h_ts(tmem + kColO + half * 128, tmem + kColS + half * 128 + (uint32_t)(k * 8), dv + (uint64_t)(k * 128), idesc_pv, t || k ? 1u : 0u);
                            if (part && last(half, t)) tc_commit(&v_free[st]);
                        }
                    }
                    ++np[half];
                    if (t + 1 < u[half]) qk(half, t + 1);
                    else if (elect_one()) tc_commit(&o_done[half]);
                }
            }
            // what this warp's tile does not see is given back all the same, when it has come
            for (int t = mine; t < units; ++t) {
                const int st = (n + t) % kStages;
                wait(&k_full[st], ph(t), 1);
                if (elect_one()) tc_commit(&k_free[st]);
                wait(&v_full[st], ph(t), 2);
                if (elect_one()) tc_commit(&v_free[st]);
            }
            n += units;
        }
        __syncwarp();
        if (abort_flag) linger();
    } else {
        // ================= softmax ===============================================================================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs<WIDENS>));
        const int half = warp >> 2, quad = warp & 3, D = a.c.D;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t s_addr = tmem + kColS + half * 128 + lanes, o_addr = tmem + kColO + half * 128 + lanes;
        uint32_t n = 0, ns = 0, no = 0, number = 0;  // tiles of keys, of scores; tiles of rows, twice
        int4 cut = make_int4(0, 0, 0, -1);
        const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.q_stride * 2) | (uintptr_t)(a.out_stride * 2)) & 15) == 0;
        for (; more; more = run.next(), ++number) {
            const Tile w = run.at();
            const long long rows = (long long)w.s.n * a.group;
            const int r = half * 128 + quad * 32 + lane;                     // row of the block's tile
            const long long row = (long long)w.tile * kRows + r;
            const bool mine = row < rows;
            const long long wfirst = row - lane;
            const long long t = w.s.first + row / a.group;
            const long long col = (long long)(w.head * a.group + (int)(row % a.group)) * D;
            const int u0 = units_of(w, 0), u1 = units_of(w, 1), units = half ? u1 : u0;
            const bool tile_there = (long long)w.tile * kRows + 128 * half < rows;
            // ---- the rows of Q: DP / 8 lanes a row ------------------------------------------------------------
            constexpr int CH = DP / 8, PER = 32 / CH;
            const int c = lane % CH;
            uint8_t *q_at = q_s + half * C::kQTile + (c / 8) * (128 * 128);
            const long long q_off = t * a.q_stride + col, out_off = t * a.out_stride + col;
            if (tile_there) {
                uint4 in[32 / PER];                                          // (all on their way at once)
#pragma unroll
                for (int i = 0; i < 32 / PER; ++i) {
                    const int rr = lane / CH + PER * i;                      // row of the warp
                    const T *src = static_cast<const T *>(a.q) + __shfl_sync(0xffffffffu, q_off, rr) + c * 8;
                    in[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (wfirst + rr < rows && c * 8 < D) {
                        if (vec) {
                            in[i] = __ldg(reinterpret_cast<const uint4 *>(src));
                        } else {
                            uint32_t y[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) y[e] = __bfloat16_as_ushort(src[2 * e]) | (uint32_t)__bfloat16_as_ushort(src[2 * e + 1]) << 16;
                            in[i] = make_uint4(y[0], y[1], y[2], y[3]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 32 / PER; ++i) {
                    const int rr = lane / CH + PER * i;
                    uint4 x = in[i];
                    if constexpr (CODED) {
                        // to fp16, the largest of the row to [2^14, 2^15): exact down to 2^-28 of it
                        float v[8];
                        unpack(x, v, T());
                        float most = 0.0f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
#pragma unroll
                        for (int o = 1; o < CH; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                        const float up = row_unit(most);
                        x = make_uint4(half2_of(v[0] * up, v[1] * up), half2_of(v[2] * up, v[3] * up), half2_of(v[4] * up, v[5] * up), half2_of(v[6] * up, v[7] * up));
                        if (c == 0) q_unit[half * 128 + quad * 32 + rr] = pow2_inverse(up);
                    }
                    *reinterpret_cast<uint4 *>(q_at + sw128(quad * 32 + rr, c % 8)) = x;
                }
                proxy_fence();
            }
            __syncwarp();
            const float row_factor = CODED && tile_there ? a.cscale * q_unit[CODED ? half * 128 + quad * 32 + lane : 0] : a.cscale;
            arrive(&q_full[half]);
            const int limit = mine ? limit_of(a, w.s, (int)row) : 0;
            const int least_limit = wfirst < rows ? limit_of(a, w.s, (int)wfirst) : 1 << 30;       // (rows behind the last: their results are not looked at)
            float m = -INFINITY, l = 0.0f;
            // Where a long run's sums are kept, and behind them their reference maximum: the place of its part, or where the tile is whole, that of the tile that goes on behind the run, the last
            // of all.  Column after column, so that the lanes' rows lie beside each other.  (Worked out when it is needed: what lives through the loop costs it registers.)
            auto place = [&] {
                const int part = run.part();
                return a.parts + (size_t)(part >= 0 ? part : 2 * (int)blockIdx.x + 1) * kRows * (DP + 2) + r;
            };
            auto factor_of = [&](const float *kept) { return kept[DP * kRows] == -INFINITY ? 0.0f : ex2_approx(kept[DP * kRows] - m); };
            for (int i0 = 0; i0 < units; i0 += kKept) {
                if (i0 > 0) {
                    wait(&s_full[half], ns & 1, 4);  // (what was summed before has come: its products were issued before those of these scores)
                    tc_fence_after();
                    float *const kept = place();
                    const float f = i0 > kKept ? factor_of(kept) : 0.0f;
#pragma unroll 1
                    for (int hh = 0; hh < DP / 16; ++hh) {
                        float x[16];
                        tmem_ld16(o_addr + hh * 16, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            float *at = kept + (hh * 16 + c) * kRows;
                            *at = i0 > kKept ? fmaf(*at, f, x[c]) : x[c];
                            x[c] = 0.0f;
                        }
                        tmem_st16(o_addr + hh * 16, x);
                    }
                    kept[DP * kRows] = m;
                    tmem_wait_st();
                }
                for (int i = i0; i < min(units, i0 + kKept); ++i) {
                    const int st = (n + i) % kStages, tb = (n + i) % kTables, p0 = (w.from + i) * kKeys;
                    wait(&s_full[half], ns++ & 1, 4);
                    tc_fence_after();
                    const uint32_t there = *reinterpret_cast<volatile uint32_t *>(&there_s[tb]);
                    const bool masked = p0 + kKeys > least_limit || there != 255u;
                    float v[4][32];
                    if constexpr (WIDENED) wait(&v_full[st], ((n + i) / kStages) & 1, 2);                  // (what was divided out comes with the values)
                    if constexpr (!SCALED) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) tmem_ld32(s_addr + q * 32, v[q]);
                        tmem_wait_ld();
                    } else {
                        // times the scales of their keys; those of 32 come while the scores do
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            float4 f[8];
                            tmem_ld32(s_addr + q * 32, v[q]);
#pragma unroll
                            for (int c = 0; c < 8; ++c) f[c] = *reinterpret_cast<const float4 *>(&ks_s[tb][q * 32 + c * 4]);
                            tmem_wait_ld();
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                const float2 lo = fmul2(make_float2(v[q][4 * c], v[q][4 * c + 1]), make_float2(f[c].x, f[c].y)), hi = fmul2(make_float2(v[q][4 * c + 2], v[q][4 * c + 3]), make_float2(f[c].z, f[c].w));
                                v[q][4 * c] = lo.x; v[q][4 * c + 1] = lo.y; v[q][4 * c + 2] = hi.x; v[q][4 * c + 3] = hi.y;
                            }
                        }
                    }
                    if (masked) {
#pragma unroll
                        for (int c = 0; c < kKeys; ++c) v[c / 32][c % 32] = p0 + c < limit && (there >> (c >> 4) & 1) ? v[c / 32][c % 32] : -INFINITY;
                    }
                    // what the scores of each 64 keys are multiplied by, and (codes) the exponent that their values were divided by: P takes it
                    float factor[2] = {row_factor, row_factor}, up[2] = {0.0f, 0.0f};
                    bool drop = false;
                    if constexpr (CODED) {
                        if constexpr (!WIDENED) wait(&v_full[st], ((n + i) / kStages) & 1, 2);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {    // (a masked score times 0 would be NaN)
                            factor[h] = fminf(fmaxf(factor[h] * *reinterpret_cast<volatile float *>(&k_unit[tb][h]), 1.17549435e-38f), 3.402823466e38f);
                            up[h] = *reinterpret_cast<volatile float *>(&v_exp[tb][h]);
                        }
                        // (values that are nothing beside the tile's others: their P, over their own power of two, would be lost, and with it their share of the sum)
                        drop = up[1] - up[0] > 60.0f;
                        if (drop) up[0] = up[1] - 60.0f;
                    }
                    float mx = -INFINITY;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 64 * h; c < 64 * h + 64; c += 2) top[c / 2 % 4] = max3(top[c / 2 % 4], v[c / 32][c % 32], v[c / 32][c % 32 + 1]);
                        mx = fmaxf(mx, fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), factor[h], up[h]));
                    }
                    if (i == 0) {
                        m = mx;
                    } else {
                        const bool grow = m == -INFINITY ? mx > m : mx > m + kRescaleStep;
                        if (__any_sync(0xffffffffu, grow)) {
                            // (codes: the maximum follows the values' exponents too, and the sum of probabilities, which does not, must not be lost where they jump: half the way twice)
                            const float step = grow ? ex2_approx(CODED ? 0.5f * (m - mx) : m - mx) : 1.0f, alpha = CODED ? step * step : step;
                            if (grow) m = mx;
                            l = CODED ? l * step * step : l * alpha;
                            // what was summed before has come: its products were issued before those of these scores
#pragma unroll 1
                            for (int hh = 0; hh < DP / 16; ++hh) {
                                float x[16];
                                tmem_ld16(o_addr + hh * 16, x);
                                tmem_wait_ld();
#pragma unroll
                                for (int c = 0; c < 16; ++c) x[c] *= alpha;
                                tmem_st16(o_addr + hh * 16, x);
                            }
                        }
                    }
                    // (fp16: P up to 2^14, its small values too)
                    const float ref = m == -INFINITY ? 0.0f : m - kBias;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t pk[16];
                        const float2 f2 = make_float2(factor[q >> 1], factor[q >> 1]), nref = make_float2(up[q >> 1] - ref, up[q >> 1] - ref);
                        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            const float2 x = ffma2(make_float2(v[q][c], v[q][c + 1]), f2, nref), y = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                            sum[c / 2 % 2] = fadd2(sum[c / 2 % 2], y);
                            pk[c / 2] = CODED ? half2_of(y.x, y.y) : pack_bf16(y.x, y.y);
                        }
                        const float part = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                        l = CODED ? fmaf(part, __uint_as_float((uint32_t)(127 - (int)up[q >> 1]) << 23), l) : l + part;
                        tmem_st16_u32(s_addr + q * 16, pk);
                        if (q == 1) {
                            if (drop) {              // (seldom)
#pragma unroll
                                for (int c = 0; c < 16; ++c) pk[c] = 0u;
                                tmem_wait_st();
                                tmem_st16_u32(s_addr, pk);
                                tmem_st16_u32(s_addr + 16, pk);
                            }
                            tmem_wait_st();
                            tc_fence_before();
                            arrive(&p_full[half][0]);
                        }
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    arrive(&p_full[half][1]);
                }
            }
            n += max(u0, u1);
            // ---- the tile's end ---------------------------------------------------------------------------------
            const int part = run.part();
            if (part >= 0 && (part & 1)) cut = run.cut();
            wait(&o_done[half], no++ & 1, 6);
            tc_fence_after();
            if (!tile_there) continue;
            const bool store = !abort_flag;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            bool wild = false;
            if (units > kKept) {
                const float *const kept = place();
                const float f = factor_of(kept);
#pragma unroll 1
                for (int hh = 0; hh < DP / 16; ++hh) {
                    float x[16];
                    tmem_ld16(o_addr + hh * 16, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = fmaf(kept[(hh * 16 + e) * kRows], f, x[e]);
                    tmem_st16(o_addr + hh * 16, x);
                }
                tmem_wait_st();
            }
            if (part >= 0) {
                float *dst = a.parts + (size_t)part * kRows * (DP + 2) + r;
#pragma unroll 1
                for (int hh = 0; hh < DP / 16; ++hh) {
                    float x[16];
                    tmem_ld16(o_addr + hh * 16, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) if (store) dst[(hh * 16 + e) * kRows] = units > 0 ? x[e] : 0.0f;
                }
                if (store) {
                    dst[DP * kRows] = m == -INFINITY ? m : m - kBias;
                    dst[(DP + 1) * kRows] = l;
                }
            } else {
                // whole rows leave by way of the tile of Q, which the last Q K^T has read
                uint8_t *turn = q_s + half * C::kQTile;
#pragma unroll 1
                for (int hh = 0; hh < DP / 16; ++hh) {
                    float x[16];
                    tmem_ld16(o_addr + hh * 16, x);
                    tmem_wait_ld();
                    uint32_t y[8];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        x[e] = l == 0.0f ? 0.0f : x[e] * inv;
                        wild = wild || (!finite(x[e]) && l == l);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
                    uint8_t *at = turn + (hh / 4) * (128 * 128);
                    *reinterpret_cast<uint4 *>(at + sw128(quad * 32 + lane, hh % 4 * 2)) = make_uint4(y[0], y[1], y[2], y[3]);
                    *reinterpret_cast<uint4 *>(at + sw128(quad * 32 + lane, hh % 4 * 2 + 1)) = make_uint4(y[4], y[5], y[6], y[7]);
                }
                __syncwarp();
#pragma unroll 4
                for (int i = 0; i < 32 / PER; ++i) {
                    const int rr = lane / CH + PER * i;
                    T *out = static_cast<T *>(a.out) + __shfl_sync(0xffffffffu, out_off, rr) + c * 8;
                    if (store && wfirst + rr < rows && c * 8 < D) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(q_at + sw128(quad * 32 + rr, c % 8));
                        if (vec) {
                            *reinterpret_cast<uint4 *>(out) = x;
                        } else {
                            const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int e = 0; e < 8; ++e) out[e] = __ushort_as_bfloat16((unsigned short)(y[e / 2] >> (e & 1) * 16));
                        }
                    }
                }
                if (__any_sync(0xffffffffu, wild && mine) && lane == 0 && store) atomicOr(&mend_s, 1u << (number & 31));
            }
            tc_fence_before();                       // (these columns are read before the next products write them)
        }
        if (tid == 0 && a.cuts) a.cuts[blockIdx.x] = cut;
        // (the other roles have come to their end, or need nothing more of this one to come to it)
        auto meet = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        meet();
        if (mend_s) mend_run<T, FMT, kRows, kKeys, kThreads>(a, &start_s, mend_s, warp, 8, tops, meet);
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && a.whole) a.whole[blockIdx.x] = !abort_flag;
    tc_fence_after();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

int encode(CUtensorMap *m, const void *rows, const cuuint64_t (&dims)[3], const cuuint64_t (&strides)[2], const cuuint32_t (&box)[3])
{
    EncodeTiledFn enc = tma_encode_fn();
    if (!enc) return fail(HIPGPT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(rows), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(HIPGPT_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
    return HIPGPT_OK;
}

// Rank-3 map {D, page size, pages * heads} over the rows of a plain 16-bit cache; a box is [1][keys of one page, 128 at most][64 values] = rows of 128 bytes, 128-byte swizzled.  What is
// outside (values from D on, a page that is none) comes as zeros.
int page_map(CUtensorMap *m, const void *rows, const PagedView &c)
{
    const cuuint64_t size = 1ull << c.shift;
    const cuuint64_t dims[3] = {(cuuint64_t)c.D, size, (cuuint64_t)c.pages * c.heads};
    const cuuint64_t strides[2] = {(cuuint64_t)c.D * 2, size * c.D * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)(size < kKeys ? size : kKeys), 1};
    return encode(m, rows, dims, strides, box);
}

// ... and over widened rows
int wide_map(CUtensorMap *m, const void *rows, const Wide &wide, const PagedView &c)
{
    const cuuint64_t dims[3] = {(cuuint64_t)c.D, (cuuint64_t)wide.room, (cuuint64_t)c.B * c.heads};
    const cuuint64_t strides[2] = {(cuuint64_t)c.D * 2, (cuuint64_t)wide.room * c.D * 2};
    const cuuint32_t box[3] = {64, kKeys, 1};
    return encode(m, rows, dims, strides, box);
}

// Codes of 64 keys of a sequence and head to fp16, as the widening warps of the kernel above do it: one read of the codes instead of one for each 256 rows of queries.  What lies behind the
// last key or in a page that is none becomes zeros; a sequence's first 128 keys are always written (a tile without keys has one unit all the same).
// Bound: memory (a byte read, two written for each code), and the chain page -> row before it: 32768 keys of 8 heads of 128, K and V: 55 us, 3.7 TB/s.
template <int FMT>
__global__ void __launch_bounds__(256)
paged_widen_kernel(const PagedView c, const Wide wide)
{
    constexpr bool SCALED = FMT == HIPGPT_CACHE_INT8;
    __shared__ float scale_s[2][kHalf], down_s[2];
    dependency_wait();
    dependents_may_start();
    const int tid = threadIdx.x, lane = tid & 31, groups = wide.room / kHalf;
    const int g = blockIdx.x % groups, bh = blockIdx.x / groups, b = bh / c.heads, head = bh % c.heads, p0 = g * kHalf;
    const Sequence s = sequence_of(c, b);
    if (s.n == 0 || p0 >= max((s.len + kKeys - 1) / kKeys, 1) * kKeys) return;
    auto row = [&](int key) { return p0 + key < s.len ? row_of(c, b, head, p0 + key) : -1LL; };
    if (tid < 64) {
        const int which = tid >> 5;
        uint32_t most = 0;
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long long at = row(lane + 32 * i);
            f[i] = at >= 0 ? (which ? c.vs : c.ks)[at] : 0.0f;
            const uint32_t bits = __float_as_uint(f[i]);
            most = max(most, bits < 0x7F800000u ? bits : 0u);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        // (values: a tile of zeros must not carry the sum of exponentials out of fp32)
        const int e = min(max((int)(most >> 23) - 127 - kUp<FMT>, which ? -96 : -126), 120);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            scale_s[which][lane + 32 * i] = SCALED && !which ? 1.0f : f[i];
            if (SCALED && !which) wide.scale[(size_t)bh * wide.room + p0 + lane + 32 * i] = f[i] * down;
        }
        if (lane == 0) {
            down_s[which] = SCALED && !which ? 1.0f : down;
            if (which) wide.v_exp[(size_t)bh * groups + g] = (float)e;
            else wide.k_unit[(size_t)bh * groups + g] = __uint_as_float((uint32_t)(127 + e) << 23);
        }
    }
    __syncthreads();
    const int chunks = c.D / 16, all = 2 * kHalf * chunks;           // of 16 codes
    uint4 raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int x = tid + 256 * i, j = x % (all / 2), which = x / (all / 2);
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (x >= all) continue;
        const long long at = row(j / chunks);
        if (at >= 0) raw[i] = __ldg(reinterpret_cast<const uint4 *>((which ? c.v : c.k) + at * c.D) + j % chunks);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int x = tid + 256 * i, j = x % (all / 2), which = x / (all / 2);
        if (x >= all) continue;
        const float f = scale_s[which][j / chunks] * down_s[which];
        const uint32_t in[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w}, f2 = half2_of(f, f);
        uint32_t out[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            codes_to_half<FMT>(in[q], out[2 * q], out[2 * q + 1]);
            out[2 * q] = mul_f16x2(out[2 * q], f2);
            out[2 * q + 1] = mul_f16x2(out[2 * q + 1], f2);
        }
        uint4 *dst = static_cast<uint4 *>(which ? wide.v : wide.k) + (((size_t)bh * wide.room + p0) * chunks + j) * 2;
        dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
        dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
}

// Joins the parts of the tile that began in this block of the kernel before and went on; a thread a row and sixteen columns, parts in ascending order.
template <int FMT, int DP>
__global__ void __launch_bounds__(256)
paged_tc_join_kernel(const __grid_constant__ AttnArgs a)
{
    using T = __nv_bfloat16;
    dependency_wait();
    dependents_may_start();
    const int4 cut = a.cuts[blockIdx.x];
    if (cut.w < 0) return;
    for (int blk = blockIdx.x; blk <= cut.w; ++blk) if (!a.whole[blk]) return;
    __shared__ int tops[8];
    const Sequence s = sequence_of(a.c, cut.x);
    const int r = threadIdx.x, D = a.c.D, c0 = blockIdx.y * 16;
    const long long row = (long long)cut.z * kRows + r, rows = (long long)s.n * a.group;
    float m = -INFINITY, l = 0.0f, o[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = 0.0f;
    if (row < rows) {
        for (int blk = blockIdx.x; blk <= cut.w; ++blk) {
            const float *p = a.parts + (size_t)(2 * blk + (blk == (int)blockIdx.x)) * kRows * (DP + 2) + r;
            float x[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = p[(c0 + e) * kRows];
            const float m2 = p[DP * kRows], l2 = p[(DP + 1) * kRows], mn = fmaxf(m, m2), base = mn == -INFINITY ? 0.0f : mn;
            // (codes: the sums of probabilities go half the way twice, as in the kernel before)
            constexpr bool CODED = FMT != HIPGPT_CACHE_PLAIN;
            const float s1 = ex2_approx(CODED ? 0.5f * (m - base) : m - base), s2 = ex2_approx(CODED ? 0.5f * (m2 - base) : m2 - base);
            const float f1 = CODED ? s1 * s1 : s1, f2 = CODED ? s2 * s2 : s2;
            m = mn;
            l = CODED ? fmaf(l * s1, s1, l2 * s2 * s2) : fmaf(l, f1, l2 * f2);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = fmaf(o[e], f1, x[e] * f2);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *out = static_cast<T *>(a.out) + (s.first + row / a.group) * a.out_stride + (long long)(cut.y * a.group + (int)(row % a.group)) * D + c0;
    bool wild = false;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        o[e] = l == 0.0f ? 0.0f : o[e] * inv;
        wild = wild || (!finite(o[e]) && l == l);
    }
    if (row < rows && c0 < D) {
        if (((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.out_stride * 2)) & 15) == 0) {
            float x[8], y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) { x[e] = o[e]; y[e] = o[8 + e]; }
            store_values<T, 8>(out, x);
            store_values<T, 8>(out + 8, y);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) out[e] = from_float<T>(o[e]);
        }
    }
    if (__syncthreads_or(row < rows && wild)) {
        const int warp = r >> 5;
        mend_tile<T, FMT, kRows>(a, cut.x, cut.y, cut.z, s, warp, 8, warp, 8, tops, [] { __syncthreads(); }, c0, c0 + 16);
    }
}

// Codes are widened before the attention, into a buffer, where the keys serve many tiles of rows and that takes at most kMostWide bytes; without the memory, in the kernel as ever.
// 16 heads over 4 of 128 in 32768 keys, int8, before / in the kernel: 512 rows a sequence 124 / 103 us, 1024 154 / 149, 2048 217 / 252, 4096 348 / 447, 16384 1069 / 1552; e4m3: 108 / 96,
// 132 / 136, 188 / 224, 297 / 399, 920 / 1393; four sequences of up to 4096 keys, int8: 1024 rows 90 / 79, 2048 121 / 125, 4096 174 / 201, 16384 551 / 637.
constexpr size_t kMostWide = (size_t)1 << 30;
constexpr long long kWideRows = 1536;
constexpr int kNoMemory = 1;             // (no status code of the library)
size_t wide_bytes(const PagedView &c, long long room) { return (size_t)c.B * c.heads * room * (4 * (size_t)c.D + 4) + (size_t)c.B * c.heads * (room / kHalf) * 8; }
// rows of the table, to whole tiles of keys
long long wide_room(const PagedView &c) { return ((((long long)c.most_pages << c.shift) + kKeys - 1) / kKeys) * kKeys; }

template <int FMT, int DP, bool WIDENED>
int launch_tc(AttnArgs a, cudaStream_t st)
{
    using C = TcCfg<FMT, DP, WIDENED>;
    const auto kern = paged_tc_kernel<FMT, DP, WIDENED>;
    // more than half of an SM's shared memory: one block an SM, for its TMEM
    constexpr size_t smem = C::kBytes > 120 * 1024 ? C::kBytes : 120 * 1024;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    static std::atomic<unsigned long long> done{0};
    if (e == cudaSuccess) e = once_per_device(done, dev, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); });
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "paged attention: %s", cudaGetErrorString(e));
    const long long room = (long long)a.c.most_pages << a.c.shift;
    const long long most = (room + kKeys - 1) / kKeys > 1 ? (room + kKeys - 1) / kKeys : 1;
    const long long tiles = ((long long)a.c.T * a.group / kRows + (a.c.T < a.c.B ? a.c.T : a.c.B)) * a.c.heads;
    int grid = sms;
    if (tiles < (1LL << 40) / most && tiles * most < grid) grid = (int)(tiles * most);
    const bool cuts = most > 1;
    StreamWorkspace::Lease ws;
    Wide wide = {};
    const size_t parts = cuts ? (size_t)2 * grid * kRows * (DP + 2) * sizeof(float) : 0, lists = cuts ? ((size_t)grid * (sizeof(int4) + sizeof(int)) + 255) / 256 * 256 : 0;
    if (cuts || WIDENED) {
        wide.room = WIDENED ? (int)wide_room(a.c) : 0;
        const int rc = g_paged_ws.enter(st, parts + lists + (WIDENED ? wide_bytes(a.c, wide.room) : 0), &ws);
        if (rc != HIPGPT_OK && WIDENED) {
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
    CUtensorMap kmap = {}, vmap = {};
    if constexpr (FMT == HIPGPT_CACHE_PLAIN) {
        int rc = page_map(&kmap, a.c.k, a.c);
        if (rc == HIPGPT_OK) rc = page_map(&vmap, a.c.v, a.c);
        if (rc != HIPGPT_OK) return rc;
    }
    if constexpr (WIDENED) {
        const size_t lots = (size_t)a.c.B * a.c.heads, each = lots * wide.room * a.c.D * 2;
        uint8_t *at = ws.get() + parts + lists;
        wide.k = at;
        wide.v = at + each;
        wide.scale = reinterpret_cast<float *>(at + 2 * each);
        wide.k_unit = wide.scale + lots * wide.room;
        wide.v_exp = wide.k_unit + lots * (wide.room / kHalf);
        int rc = wide_map(&kmap, wide.k, wide, a.c);
        if (rc == HIPGPT_OK) rc = wide_map(&vmap, wide.v, wide, a.c);
        if (rc != HIPGPT_OK) return rc;
        e = launch_overlapped(paged_widen_kernel<FMT>, dim3((unsigned)(lots * (wide.room / kHalf))), dim3(256), 0, st, a.c, wide);
        if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "paged_widen_kernel: %s", cudaGetErrorString(e));
    }
    e = launch_overlapped(kern, dim3((unsigned)grid), dim3(kThreads), smem, st, kmap, vmap, a, wide, take_expiry(1000));
    if (e == cudaSuccess && cuts) e = launch_overlapped(paged_tc_join_kernel<FMT, DP>, dim3((unsigned)grid, DP / 16), dim3(kRows), 0, st, a);
    return e == cudaSuccess ? check_launch("paged_tc_kernel") : fail(HIPGPT_ERR_CUDA, "paged_tc_kernel: %s", cudaGetErrorString(e));
}

}  // namespace

int launch_paged_tc(int format, const AttnArgs &a, cudaStream_t st)
{
    const bool narrow = a.c.D <= 64;
    if (format == HIPGPT_CACHE_PLAIN) return narrow ? launch_tc<HIPGPT_CACHE_PLAIN, 64, false>(a, st) : launch_tc<HIPGPT_CACHE_PLAIN, 128, false>(a, st);
    const long long room = wide_room(a.c);
    const bool wide = room > 0 && (long long)a.c.T * a.group >= kWideRows * a.c.B && (long long)a.c.heads * a.c.B <= (long long)(kMostWide / 64) / room && wide_bytes(a.c, room) <= kMostWide;
    if (wide) {
        const int rc = format == HIPGPT_CACHE_E4M3 ? (narrow ? launch_tc<HIPGPT_CACHE_E4M3, 64, true>(a, st) : launch_tc<HIPGPT_CACHE_E4M3, 128, true>(a, st))
                                                   : (narrow ? launch_tc<HIPGPT_CACHE_INT8, 64, true>(a, st) : launch_tc<HIPGPT_CACHE_INT8, 128, true>(a, st));
        if (rc != kNoMemory) return rc;
    }
    if (format == HIPGPT_CACHE_E4M3) return narrow ? launch_tc<HIPGPT_CACHE_E4M3, 64, false>(a, st) : launch_tc<HIPGPT_CACHE_E4M3, 128, false>(a, st);
    return narrow ? launch_tc<HIPGPT_CACHE_INT8, 64, false>(a, st) : launch_tc<HIPGPT_CACHE_INT8, 128, false>(a, st);
}

int paged_status_fetch(int *status)
{
    int s = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&s, g_paged_status, sizeof(int));
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "cudaMemcpyFromSymbol: %s", cudaGetErrorString(e));
    if (s != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_paged_status, &zero, sizeof(int));
    }
    *status = s;
    return HIPGPT_OK;
}

}  // namespace hipgpt
