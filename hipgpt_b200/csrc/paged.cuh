// A cache in pages and the ragged batch that works on it: what rotary.cu, paged_cache.cu, attn_paged.cu and attn_paged_tc.cu share.
//
//   cache   k, v [pages][heads][page size][D] of the activations' type, or of 8-bit codes with one fp32 scale per row ([pages][heads][page size])
//   batch   sequence b's new tokens are the rows offsets[b] .. offsets[b+1] of the call's tensors; they are the last of the lengths[b] tokens that the
//           sequence has with them; position p of it lies in page table[b][p / page size], at p % page size
//
// What the device holds is not known to the host and is not trusted: offsets are cut to [0, T], lengths to what a row of the table can hold, and a page
// number outside the cache is a page without tokens.
#pragma once

#include "elem_types.cuh"

namespace hipgpt {

struct PagedView {
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int *offsets, *lengths, *table;
    int B, T, most_pages, pages, shift, heads, D;
};

struct Sequence { int first, n, len; };          // first row, new tokens, length with them
__device__ __forceinline__ Sequence sequence_of(const PagedView &c, int b)
{
    const int a = min(max(__ldg(c.offsets + b), 0), c.T), e = min(max(__ldg(c.offsets + b + 1), 0), c.T);
    const long long room = (long long)c.most_pages << c.shift;
    return {a, max(e - a, 0), (int)min((long long)max(__ldg(c.lengths + b), 0), room)};
}

// The row of position p (>= 0, below the sequence's length) of sequence b in units of rows of the cache, -1 where its page is none
__device__ __forceinline__ long long row_of(const PagedView &c, int b, int head, int p)
{
    const int page = __ldg(c.table + (size_t)b * c.most_pages + (p >> c.shift));
    if (page < 0 || page >= c.pages) return -1;
    return ((((long long)page * c.heads) + head) << c.shift) + (p & ((1 << c.shift) - 1));
}

// ---- 8-bit codes as fp16 (exact; NaN codes of e4m3 are NaN, in attention and when read back) ----
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) { uint32_t r; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo)); return r; }
__device__ __forceinline__ float2 floats_of(uint32_t half2)
{
    float2 f;
    asm("{.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tcvt.f32.f16 %0, x;\n\tcvt.f32.f16 %1, y;}" : "=f"(f.x), "=f"(f.y) : "r"(half2));
    return f;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) { uint32_t r; asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
// Four codes of a word, in two words
template <int FMT>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi)
{
    if constexpr (FMT == HIPGPT_CACHE_E4M3) {
        asm("{.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        w ^= 0x80808080u;                            // 128 more, without sign; 0x64 above a byte u is 1024 + u
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(__byte_perm(w, 0x64646464u, 0x4140)), "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(__byte_perm(w, 0x64646464u, 0x4342)), "r"(0x64806480u));
    }
}

// What the host checks of a cache and a batch (0: go on, 1: nothing to do, < 0: refused)
inline int check_paged(const hipgpt_paged_cache *c, const hipgpt_paged_batch *b, PagedView *out)
{
    if (!c || !b) return fail(HIPGPT_ERR_NULL, "cache and batch must not be NULL");
    if (c->type != HIPGPT_TYPE_F32 && c->type != HIPGPT_TYPE_BF16) return fail(HIPGPT_ERR_BAD_ARG, "unknown type %d", c->type);
    if (c->format != HIPGPT_CACHE_PLAIN && c->format != HIPGPT_CACHE_E4M3 && c->format != HIPGPT_CACHE_INT8) return fail(HIPGPT_ERR_BAD_ARG, "unknown cache format %d", c->format);
    if (c->pages < 0 || c->heads <= 0 || c->head_dim <= 0 || b->sequences < 0 || b->tokens < 0 || b->most_pages < 0)
        return fail(HIPGPT_ERR_BAD_ARG, "bad size: pages=%d heads=%d head_dim=%d sequences=%d tokens=%d most_pages=%d", c->pages, c->heads, c->head_dim, b->sequences, b->tokens, b->most_pages);
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) return fail(HIPGPT_ERR_BAD_ARG, "page size %d is no power of two from 16 to 1024", c->page_size);
    if (c->head_dim % 16 || c->head_dim > 128) return fail(HIPGPT_ERR_UNSUPPORTED, "head_dim %d is no multiple of 16 up to 128", c->head_dim);
    if ((long long)c->heads * c->head_dim > 1 << 24) return fail(HIPGPT_ERR_BAD_ARG, "rows of %d heads of %d values are too long", c->heads, c->head_dim);
    if ((long long)b->most_pages * c->page_size > 1 << 30) return fail(HIPGPT_ERR_BAD_ARG, "%d pages of %d tokens are beyond one sequence", b->most_pages, c->page_size);
    if ((long long)c->pages * c->heads > 2147483646LL || (long long)c->pages * c->heads * c->page_size > 1LL << 40) return fail(HIPGPT_ERR_BAD_ARG, "a cache of %d pages is too large", c->pages);
    if (b->tokens == 0 || b->sequences == 0) return 1;
    if (!b->offsets || !b->lengths || (!b->page_table && b->most_pages > 0)) return fail(HIPGPT_ERR_NULL, "offsets, lengths and the page table must not be NULL");
    const bool coded = c->format != HIPGPT_CACHE_PLAIN;
    if (c->pages > 0 && (!c->k || !c->v || (coded && (!c->k_scale || !c->v_scale)))) return fail(HIPGPT_ERR_NULL, "the cache's arrays must not be NULL");
    if (!all_aligned16({c->k, c->v, c->k_scale, c->v_scale})) return fail(HIPGPT_ERR_BAD_ARG, "the cache's arrays must start on 16-byte boundaries");
    int shift = 0;
    while ((1 << shift) < c->page_size) ++shift;
    *out = {static_cast<const uint8_t *>(c->k), static_cast<const uint8_t *>(c->v), c->k_scale, c->v_scale, b->offsets, b->lengths, b->page_table,
            b->sequences, b->tokens, b->most_pages, c->pages, shift, c->heads, c->head_dim};
    return HIPGPT_OK;
}

inline size_t cache_element_bytes(const hipgpt_paged_cache *c) { return c->format != HIPGPT_CACHE_PLAIN ? 1 : c->type == HIPGPT_TYPE_F32 ? 4 : 2; }
inline size_t cache_rows(const hipgpt_paged_cache *c) { return (size_t)c->pages * c->heads * c->page_size; }

// Rows of `width` bytes, `stride` bytes apart
struct Rows { const void *at; size_t stride, width; long long n; };
inline size_t extent_of(const Rows &r) { return r.n > 0 ? (size_t)(r.n - 1) * r.stride + r.width : 0; }
// Columns of one wider array (the same stride) may lie beside each other; otherwise what is between the rows counts as theirs
inline bool rows_overlap(const Rows &a, const Rows &b)
{
    if (!a.at || !b.at || a.n <= 0 || b.n <= 0 || !ranges_overlap(a.at, extent_of(a), b.at, extent_of(b))) return false;
    if (a.stride != b.stride) return true;
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a.at), pb = reinterpret_cast<uintptr_t>(b.at);
    const size_t d = pb >= pa ? (pb - pa) % a.stride : (a.stride - (pa - pb) % a.stride) % a.stride;
    return !(d >= a.width && d + b.width <= a.stride);
}
inline int check_stride(const char *what, long long stride, long long width)
{
    if (stride < width || stride > 1LL << 40) return fail(HIPGPT_ERR_BAD_ARG, "%s: rows of %lld values cannot be %lld apart", what, width, stride);
    return HIPGPT_OK;
}
// A written array against the batch's and the cache's
inline int refuse_rows_over(const Rows &out, std::initializer_list<Rows> others, const hipgpt_paged_cache *c, const hipgpt_paged_batch *b)
{
    for (const Rows &o : others) if (rows_overlap(out, o)) return fail(HIPGPT_ERR_BAD_ARG, "an output overlaps another of the call's arrays");
    const size_t rows = cache_rows(c), bytes = rows * c->head_dim * cache_element_bytes(c);
    for (const Extent &e : {Extent{c->k, bytes}, Extent{c->v, bytes}, Extent{c->k_scale, rows * 4}, Extent{c->v_scale, rows * 4}, Extent{b->offsets, 4 * ((size_t)b->sequences + 1)},
                            Extent{b->lengths, 4 * (size_t)b->sequences}, Extent{b->page_table, 4 * (size_t)b->sequences * b->most_pages}})
        if (e.at && e.bytes && out.at && ranges_overlap(out.at, extent_of(out), e.at, e.bytes)) return fail(HIPGPT_ERR_BAD_ARG, "an output overlaps another of the call's arrays");
    return HIPGPT_OK;
}

}  // namespace hipgpt
