// What the kernels over a paged key-value cache share: where a row lives, which sequence a packed token belongs to, rotary
// angles that stay exact at far positions, and the host's checks of the cache's geometry.
//
// The cache is [num_layers, num_pages, Hkv, page_size, D]: the rows of one kv head inside one page are contiguous
// (page_size * D elements), so a tile of 16 rows is one contiguous block - page_size is a power of two of 16 or more, and
// everything below walks the rows in aligned groups of 16, each of which lies in one page.
#pragma once
#include <math.h>
#include "common.hpp"
#include "rope.hpp"

namespace onellm {

constexpr int kPagedMaxD = 256;                // head sizes the paged kernels are built for
constexpr int kRowGroup = 16;                  // rows that are known to share a page

struct PagedCache {
    const int* table;      // [B, max_pages]
    int max_pages, num_pages, page_shift;
    int Hkv, D;
    size_t slab;           // element offset of the layer inside the page array
};

// The page that holds row `row` of a sequence, -1 where there is none: a row past the table's end, or an entry that
// names no page of the array.
__device__ __forceinline__ int page_of(const PagedCache& c, const int* table_row, int row)
{
    const int p = row >> c.page_shift;
    if (p >= c.max_pages) return -1;
    // (nothing writes the table while a kernel runs: read as constant memory, by the scalar unit where p is uniform)
    typedef const __attribute__((address_space(4))) int const_int;
    const int id = ((const_int*)reinterpret_cast<uintptr_t>(table_row))[p];
    return (unsigned)id < (unsigned)c.num_pages ? id : -1;
}

// rows of the group at row0 that lie in front of `end` (both the same in every lane; the three-operand clamp only exists on the
// vector unit, so its result is brought back to a scalar register: a memory window has to be one)
__device__ __forceinline__ int rows_left(int end, int row0)
{
    return __builtin_amdgcn_readfirstlane(min(max(end - row0, 0), kRowGroup));
}

// element offset of row `row` (of the sequence) of kv head `kvh` in page `page`
__device__ __forceinline__ size_t paged_offset(const PagedCache& c, int page, int kvh, int row)
{
    const size_t block = (size_t)page * c.Hkv + kvh;
    return c.slab + ((block << c.page_shift) + (row & ((1 << c.page_shift) - 1))) * (size_t)c.D;
}

// Rotary tables in turns per position: the angle of pair i at position p is p * f[i] turns.  The product and its reduction
// to a fraction of a turn are done in 64 bits (off by at most 3e-14 of p * f, 2e-9 rad at position 65536), so the
// rotation of a far position is as exact as that of a near one; p / base^(2i/dim) rounded to 32 bits would be off by
// up to 2^-24 of the angle, 4e-3 rad at position 65536.
struct RopeTurns { double f[kPagedMaxD / 2]; };

// (one power per call, the rest by multiplication: 2^-52 relative per pair, 1e-14 at the last one)
inline void fill_rope_turns(RopeTurns& rt, int D, int rotary_dim, float base)
{
    constexpr double kTwoPi = 6.283185307179586476925286766559;
    const double step = rotary_dim > 0 ? pow((double)base, -2.0 / (double)rotary_dim) : 0.0;
    double f = 1.0 / kTwoPi;
    for (int i = 0; i < kPagedMaxD / 2; ++i) {
        rt.f[i] = 2 * i < rotary_dim && 2 * i + 1 < D ? f : 0.0;
        f *= step;
    }
}

__device__ __forceinline__ void rope_sincos(int pos, double turns_per_pos, float& s, float& c)
{
    const double t = (double)pos * turns_per_pos;
    const double frac = t - __builtin_rint(t);                       // [-1/2, 1/2] of a turn
    sincos_fixed((float)(frac * 6.283185307179586476925286766559), s, c);
}

inline int log2_of(int v)
{
    int s = 0;
    while ((1 << s) < v) ++s;
    return s;
}

// The host's checks of a paged call's geometry.  Everything a kernel multiplies up in 32 bits is bounded here.
inline int check_paged(int dtype, const void* k_pages, const void* v_pages, const int* block_table, int B, int Hq, int Hkv, int D,
                       int page_size, int num_pages, int max_pages, int layer, int num_layers)
{
    if (!k_pages || !v_pages || !block_table) return ONELLM_EINVAL;
    if (dtype != ONELLM_FP32 && dtype != ONELLM_FP16) return ONELLM_EINVAL;
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || Hq % Hkv != 0) return ONELLM_EINVAL;
    if (page_size <= 0 || num_pages <= 0 || max_pages <= 0) return ONELLM_EINVAL;
    if (layer < 0 || num_layers <= 0 || layer >= num_layers) return ONELLM_EINVAL;
    if (page_size < kRowGroup || (page_size & (page_size - 1)) != 0) return ONELLM_EUNSUPPORTED;
    const int vec = dtype == ONELLM_FP16 ? 8 : 4;
    if (D > kPagedMaxD || D % vec != 0) return ONELLM_EUNSUPPORTED;
    // rows of one sequence, query heads and one page's bytes stay far from the ends of 32 bits
    if ((long long)page_size * max_pages > 0x3FFFFFFFLL || B > 65535 || Hq > 4096) return ONELLM_EUNSUPPORTED;
    if ((long long)page_size * D * (16 / vec) > 0x3FFFFFFFLL) return ONELLM_EUNSUPPORTED;
    if (!aligned16(k_pages) || !aligned16(v_pages)) return ONELLM_EUNSUPPORTED;
    return 0;
}

inline PagedCache make_paged(const int* block_table, int max_pages, int num_pages, int page_size, int Hkv, int D, int layer)
{
    PagedCache c;
    c.table = block_table;
    c.max_pages = max_pages;
    c.num_pages = num_pages;
    c.page_shift = log2_of(page_size);
    c.Hkv = Hkv;
    c.D = D;
    c.slab = (size_t)layer * num_pages * Hkv * page_size * D;
    return c;
}

// Whether n rows of x_len elements and n of y_len, x_stride and y_stride elements apart, share memory.  Rows of one stride may lie
// between each other's.
inline bool rows_overlap(const void* x, long x_stride, long x_len, const void* y, long y_stride, long y_len, long n, size_t elt)
{
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(x), y0 = reinterpret_cast<uintptr_t>(y);
    const uintptr_t x1 = x0 + ((n - 1) * x_stride + x_len) * elt, y1 = y0 + ((n - 1) * y_stride + y_len) * elt;
    if (x1 <= y0 || y1 <= x0) return false;
    if (n == 1 || x_stride != y_stride) return true;
    // a row of y starts d bytes behind one of x, the next one of x a stride behind that
    const uintptr_t stride = x_stride * elt;
    const uintptr_t d = x0 <= y0 ? (y0 - x0) % stride : (stride - (x0 - y0) % stride) % stride;
    return d < x_len * elt || stride - d < y_len * elt;
}

}  // namespace onellm
