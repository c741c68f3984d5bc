// Attention of packed prompt tokens over a paged key-value cache: causal, grouped heads, sequences of different lengths.
//
//   o[i] = sum_j softmax_j(q[i] . k[j] / sqrt(D)) v[j]   over rows j <= history + i of the token's sequence
//
// One pass over the rows with a running maximum and sum.  The query heads that share a kv head and the tokens of a sequence
// are one axis (row m = token * G + head), so a tile of 128 rows reads K and V once for all of them.
//
// A wave owns 32 rows.  It computes the transposed score tile S^T = K Q^T: in the result layout of the 32 x 32 products a
// lane then holds 16 of the 32 keys' scores of ONE row (the other half is in lane ^ 32), so the softmax needs a single
// lane exchange per tile, and the registers it leaves are, as they stand, the B operand of O^T = V^T P^T: product i takes
// the keys its lanes hold, and V^T's operand picks the same keys.  For fp16 that operand (a column of V over four
// keys) comes out of the LDS transposed (ds_read_b64_tr_b16); for fp32 a product takes two keys and reads them as they are.
// Scores, statistics and output are fp32.  fp16: P enters its product rounded to fp16 (half a step, 2^-11 relative of each
// weight, averaged over the keys: together at most about what the result's own rounding adds); the sum of the weights is taken before
// that rounding.  P in two parts, 8192 tokens: 781 us instead of 574.
//
// 128 rows per workgroup: every K and V row that comes through LDS is then used for 128 products, and a wave's 32 rows of scores, output
// and Q leave room for two workgroups on a compute unit (heads up to 128), of which one multiplies while the other takes exponentials.
// Bound by that pair of units, not by memory: 8192 tokens of 32 heads on 8 of 128, fp16, 544..577 us, 950..1010 TFLOP/s (a library product
// of 16384^3 reaches 1266 on the same card), matrix cores 54 % busy and the vector unit 53 %.  2058 tokens in four sequences, fp32, 16 heads on 2
// of 64: 62.5 us.  Heads between 64, 128 and 256 are multiplied at the next of these: 8192 tokens with heads of 96 / 160 / 192 / 256 506 / 1436 /
// 1446 / 1464 us.
#include <type_traits>
#include "paged.hpp"

namespace onellm {
namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kRowsPerTile = 128, kThreads = 256;

struct PromptArgs {
    const void* q;
    const void* k_pages;
    const void* v_pages;
    void* out;
    const int* cu;
    const int* hist;
    PagedCache cache;
    long q_stride, out_stride;
    int B, token_num, Hq, G;
    float score_scale;         // log2(e) / sqrt(D)
    int nsplit;                // pieces a tile's rows of the cache are cut into
    float* part_o;             // [nsplit, token_num * Hq, D]
    float* part_ml;            // [nsplit, token_num * Hq, 2]
};

// The tile a workgroup works on.  Tiles are numbered longest first, as far as that is cheap to say: the sequences of a block of 64 by
// their rows, the tiles of a sequence from its end - workgroups start in this order, and the last ones should be short.
// (eight prompts of 1..2048 tokens in the order they came: 98 us, by length 91.)
struct Tile {
    int b, first, len, hist;   // sequence, its first packed token, tokens, rows before them
    int m0;                    // first row of the tile: token m / G, head m % G of the group
};

// sum over the lanes up to this one
__device__ __forceinline__ int wave_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);        // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);        // lane 15 of the row before, to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);        // lane 31, to rows 2 and 3
    return v;
}

__device__ __forceinline__ bool locate_tile(const PromptArgs& a, int index, Tile& t)
{
    const int lane = threadIdx.x & (kWave - 1);
    int run = 0;
    for (int c = 0; c < a.B; c += kWave) {
        const int b = c + lane;
        int first = 0, len = 0, hist = 0, n = 0;
        if (b < a.B) {
            first = max(a.cu[b], 0);
            len = min(max(a.cu[b + 1], 0), a.token_num) - first;
            hist = a.hist[b];
            if (len > 0 && hist >= 0) n = (len * a.G + kRowsPerTile - 1) / kRowsPerTile;
            hist = min(hist, 1 << 30);              // (past every table: all its rows are seen)
        }
        // rank by rows, no two alike (beyond 2^25 rows the order no longer matters)
        const int key = n > 0 ? min(hist + len, (1 << 25) - 1) * kWave + (kWave - 1 - lane) : -1 - lane;
        int rank = 0;
        for (int j0 = 0; j0 < kWave; j0 += 16) {
            if (c + j0 >= a.B) break;
#pragma unroll
            for (int j = 0; j < 16; ++j) rank += __builtin_amdgcn_readlane(key, j0 + j) > key ? 1 : 0;
        }
        if (b >= a.B) rank = lane;                  // (their keys are below all others and rank among themselves)
        // in the order of the ranks: whose turn it is, and how many tiles there are up to its last
        const int whose = __builtin_amdgcn_ds_permute(rank * 4, lane);
        const int inc = wave_scan(__builtin_amdgcn_ds_permute(rank * 4, n));
        const int tot = __builtin_amdgcn_readlane(inc, kWave - 1);
        if (index < run + tot) {
            const int f = __builtin_ctzll(__builtin_amdgcn_ballot_w64(run + inc > index));
            const int from = __builtin_amdgcn_readlane(whose, f);
            t.b = c + from;
            t.first = __builtin_amdgcn_readlane(first, from);
            t.len = __builtin_amdgcn_readlane(len, from);
            t.hist = __builtin_amdgcn_readlane(hist, from);
            t.m0 = (run + __builtin_amdgcn_readlane(inc, f) - 1 - index) * kRowsPerTile;
            return true;
        }
        run += tot;
    }
    return false;
}

constexpr unsigned kOutside = 0x7FFFFF00u;     // a byte offset no window of 16 rows reaches
constexpr float kFar = 4096.f;
constexpr float kLowest = -3.4028234664e38f;

template <typename T, int DP>
struct PromptShape {
    static constexpr bool kHalf = sizeof(T) == 2;
    static constexpr int VEC = 16 / sizeof(T);
    static constexpr int BN = kHalf && DP <= 128 ? 64 : 32; // keys per step
    static constexpr int P = DP / VEC;                      // 16-byte pieces of a staged row
    static constexpr int ROW = DP * (int)sizeof(T);         // bytes of a staged row
    static constexpr int LD = BN * P / kThreads;            // pieces per thread and operand
    static constexpr int NG = BN / kRowGroup;               // row groups per step
    static constexpr int NS = BN / 32;                      // score tiles per step
    static constexpr int ND = DP / 32;                      // output tiles
    static constexpr int TILE = BN * ROW;                   // bytes of a staged operand
    static_assert(BN * P % kThreads == 0 && (kWave / P <= kRowGroup), "whole pieces per thread; a wave's pieces lie in one row group");
    // LDS keeps piece p of row r at p ^ swizzle(r): without it the lanes of a read would all hit the same banks.  K: 16 lanes
    // of a 16-byte read take one piece each of 16 rows.  V, fp16: 32 lanes of a transposed read take 64 bytes each of four rows (a
    // swizzle that spread only the 16 lanes of one transposition cost two cycles in four); fp32: 32 columns of two rows.
    __device__ static __forceinline__ int swz_k(int r) { return P == 8 ? (r >> 1) & 7 : r & 15; }
    __device__ static __forceinline__ int swz_v(int r)
    {
        if constexpr (!kHalf) return ((r >> 2) & 1) * 8;
        else return P == 8 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
    }
};

// four consecutive elements out of a window (zeros behind its end)
template <typename T> struct Quad { T v[4]; };
template <typename T>
__device__ __forceinline__ Quad<T> load_quad(__amdgpu_buffer_rsrc_t w, int offset)
{
    if constexpr (sizeof(T) == 2) return __builtin_bit_cast(Quad<T>, __builtin_amdgcn_raw_buffer_load_b64(w, offset, 0, 0));
    else return __builtin_bit_cast(Quad<T>, __builtin_amdgcn_raw_buffer_load_b128(w, offset, 0, 0));
}

__device__ __forceinline__ float other_half_max(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <typename T, int DP>
__device__ __forceinline__ void prompt_tile(const PromptArgs& a)
{
    using S = PromptShape<T, DP>;
    constexpr int VEC = S::VEC, BN = S::BN, P = S::P, LD = S::LD, NS = S::NS, ND = S::ND;
    // (four arrays, not one: the compiler then sees that the rows on their way to one pair do not touch the other)
    __shared__ __align__(16) char k_even[S::TILE], v_even[S::TILE], k_odd[S::TILE], v_odd[S::TILE];
    __shared__ int s_odd;                           // a masked step met a NaN or an infinity in V

    Tile t;
    // (the pieces of a tile next to each other, so that the longest pieces of all start first - with the tiles of one piece after those of the
    // other, every second one in the opposite order: 461 tokens behind 15000..20000 rows 178 us, so 167; 2048 tokens fp32 366, 324)
    if (!locate_tile(a, blockIdx.z, t)) return;
    // the same in every lane: said here, behind the search's loops, so that all that follows from it stays scalar
    t.b = __builtin_amdgcn_readfirstlane(t.b);
    t.first = __builtin_amdgcn_readfirstlane(t.first);
    t.len = __builtin_amdgcn_readfirstlane(t.len);
    t.hist = __builtin_amdgcn_readfirstlane(t.hist);
    t.m0 = __builtin_amdgcn_readfirstlane(t.m0);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int kvh = blockIdx.x, D = a.cache.D;
    const int M = t.len * a.G;
    const int m = t.m0 + wave * 32 + col;           // this lane's row
    const bool row_ok = m < M;
    const int token = row_ok ? m / a.G : 0, head = kvh * a.G + (row_ok ? m % a.G : 0);
    // (a division leaves its quotient in a vector register: back to a scalar one, with all that follows from it)
    const int last = __builtin_amdgcn_readfirstlane(min((t.m0 + kRowsPerTile - 1) / a.G, t.len - 1));
    const int rows_end = min(t.hist + last + 1, a.cache.max_pages << a.cache.page_shift);       // rows any row of the tile sees
    const int rows_all = t.hist + __builtin_amdgcn_readfirstlane(t.m0 / a.G) + 1;               // rows every row of it sees
    // equal pieces of the tile's own rows, in whole steps
    const int chunk = a.nsplit == 1 ? rows_end : (__builtin_amdgcn_readfirstlane((rows_end + a.nsplit - 1) / a.nsplit) + 63) / 64 * 64;
    const int k_begin = blockIdx.y * chunk, k_end = min(k_begin + chunk, rows_end);
    const int limit = min(t.hist + token, k_end - 1);      // the last key the row sees (the table may end before its position)
    const int* table = a.cache.table + (size_t)t.b * a.cache.max_pages;

    // Q: lane (col, half) holds pieces 2 k + half of its row
    Vec16<T> qf[P / 2];
    {
        const T* q = static_cast<const T*>(a.q) + (size_t)(t.first + token) * a.q_stride + (size_t)head * D;
#pragma unroll
        for (int k = 0; k < P / 2; ++k) {
            const int p = 2 * k + half;
#pragma unroll
            for (int e = 0; e < VEC; ++e) qf[k].set(e, 0.f);
            if (row_ok && p * VEC < D) qf[k] = load16(q + p * VEC);
        }
    }

    if (tid == 0) s_odd = 0;
    int odd_from = k_begin;
    float mx = -INFINITY, l = 0.f;                  // of this lane's row: what weights are relative to; their sum over this lane's keys
    const float slack = 8.f / a.score_scale;
    bool far = false;                               // a row of the wave has a reference of 2^12 or more in units of log 2
    auto is_far = [&](float ref) __attribute__((always_inline)) { return ref != -INFINITY && __builtin_fabsf(ref * a.score_scale) >= kFar; };
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;

    // Where the rows are.  A step's rows are NG groups of 16 and every wave needs each group's address in scalar registers; looked
    // up one by one that was 240 scalar instructions per step, a third of the kernel's time.  So the lanes of a wave look
    // up 64 groups at once - lane g the g-th of a block of SPB steps - and a step reads its groups' offsets out of them.
    constexpr int SPB = kWave / S::NG;              // steps per block
    auto pages_of = [&](int block) __attribute__((always_inline)) {      // page of this lane's group, -1: none
        const int row = k_begin + (block * kWave + lane) * kRowGroup;
        const int id = table[min(row, k_end - 1) >> a.cache.page_shift];     // (k_end lies inside the table; no branch around the load)
        return row < k_end && (unsigned)id < (unsigned)a.cache.num_pages ? id : -1;
    };
    unsigned off_lo = 0, off_hi = 0;                // byte offset of this lane's group in the page arrays
    unsigned long long there = 0;                   // the groups of the block that have a page
    auto open_block = [&](int block, int page) __attribute__((always_inline)) {
        there = __builtin_amdgcn_ballot_w64(page >= 0);
        const size_t at = paged_offset(a.cache, max(page, 0), kvh, k_begin + (block * kWave + lane) * kRowGroup) * sizeof(T);
        off_lo = (unsigned)at;
        off_hi = (unsigned)(at >> 32);
    };
    // Rows k0 .. k0 + BN - 1 go straight from memory to LDS, 16 bytes per lane: slot (tid + 256 i) is (row, p') and
    // gets piece p' ^ swizzle(row).  A wave's slots lie in one group of 16 rows, which is read through a window that holds
    // the rows the sequence has there: rows behind its end, rows on a page that is none, and pieces behind the head's
    // end arrive as zeros.
    constexpr int RI = kThreads / P;                // rows between two slots of a thread
    constexpr int NOFF = RI % kRowGroup == 0 ? 1 : kRowGroup / RI;      // different places inside a window
    unsigned koff[NOFF], voff[NOFF];
#pragma unroll
    for (int i = 0; i < NOFF; ++i) {
        const int row = i * RI + tid / P, p = tid % P;
        const unsigned line = (unsigned)((row % kRowGroup) * D) * (unsigned)sizeof(T);
        const int pk = p ^ S::swz_k(row), pv = p ^ S::swz_v(row);
        koff[i] = pk * VEC < D ? line + pk * 16 : kOutside;
        voff[i] = pv * VEC < D ? line + pv * 16 : kOutside;
    }
    // EDGE: the step may reach past the sequence's end or lie on pages that are none (without it the rows are all there,
    // or stand on a page that is not looked at: a masked step leaves them out)
    auto request = [&](char* kb, char* vb, int step, auto edge_tag) __attribute__((always_inline)) {
        constexpr bool EDGE = decltype(edge_tag)::value;
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int group = step * S::NG + (i * kThreads + wave * 64) / P / kRowGroup;       // (the wave's group)
            const size_t at = (size_t)(unsigned)__builtin_amdgcn_readlane((int)off_hi, group % kWave) << 32
                              | (unsigned)__builtin_amdgcn_readlane((int)off_lo, group % kWave);
            int rows = kRowGroup;
            if constexpr (EDGE) rows = (there >> (group % kWave) & 1) ? rows_left(k_end, k_begin + group * kRowGroup) : 0;
            const int bytes = rows * D * (int)sizeof(T);
            char* kp = const_cast<char*>(static_cast<const char*>(a.k_pages)) + at;
            char* vp = const_cast<char*>(static_cast<const char*>(a.v_pages)) + at;
            typedef __attribute__((address_space(3))) void lds_void;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(kp, 0, bytes, 0x00020000),
                                                     (lds_void*)(kb + (i * kThreads + wave * 64) * 16), 16, koff[i % NOFF], 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(vp, 0, bytes, 0x00020000),
                                                     (lds_void*)(vb + (i * kThreads + wave * 64) * 16), 16, voff[i % NOFF], 0, 0, 0);
        }
    };
    // Masked steps: a NaN or an infinity in a V row would reach rows that do not see it (0 * NaN), so every thread
    // first replaces those among the pieces it brought by zeros; the rows that do see them get them behind the loop.
    // (found by their exponent bits: adding one to an exponent of all ones carries into the sign's place)
    auto clean = [&](char* vb) __attribute__((always_inline)) {
        constexpr unsigned EXP = S::kHalf ? 0x7C007C00u : 0x7F800000u, ONE = S::kHalf ? 0x04000400u : 0x00800000u;
        constexpr unsigned CARRY = S::kHalf ? 0x80008000u : 0x80000000u;
        u32x4 v[LD];
        unsigned carry = 0;
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            v[i] = *reinterpret_cast<const u32x4*>(vb + (i * kThreads + tid) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) carry |= (v[i][e] & EXP) + ONE;
        }
        if (__builtin_amdgcn_ballot_w64((carry & CARRY) != 0)) {
#pragma unroll 1
            for (int i = 0; i < LD; ++i) {
                Vec16<T>* at = reinterpret_cast<Vec16<T>*>(vb + (i * kThreads + tid) * 16);
                Vec16<T> x = *at;
#pragma unroll
                for (int e = 0; e < VEC; ++e) x.set(e, __builtin_fabsf(x.get(e)) < INFINITY ? x.get(e) : 0.f);
                *at = x;
            }
            s_odd = 1;
        }
    };

    // one step: keys k0 .. k0 + BN - 1.  valid: bit g = group g's page exists (masked steps only)
    auto compute = [&](const char* kb, const char* vb, int k0, auto masked_tag, unsigned valid) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        // Reads from LDS are issued two products ahead (K) or one group of products ahead (V); the scheduling barriers keep
        // them there - left alone, the compiler reads every operand right before its product and waits for it.
        f32x16 s[NS];
        Vec16<T> kf[P / 2][NS];
        auto read_k = [&](int k) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                const int row = n * 32 + col;
                kf[k][n].raw = *reinterpret_cast<const decltype(kf[k][n].raw)*>(kb + row * S::ROW + ((2 * k + half) ^ S::swz_k(row)) * 16);
            }
        };
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[n][r] = 0.f;
        read_k(0);
        read_k(1);
#pragma unroll
        for (int k = 0; k < P / 2; ++k) {
            if (k + 2 < P / 2) read_k(k + 2);
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                if constexpr (S::kHalf) {
                    s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k][n].raw, qf[k].raw, s[n], 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[k][n].raw[e], qf[k].raw[e], s[n], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // V^T operands.  fp16: of 16 keys, 16 i + 8 (e / 4) + 4 half + e % 4, which is what the score registers 8 (i % 2) .. + 7
        // of this lane are: 16 lanes read four rows x 16 columns, four elements each, and get one column of the four rows each.
        // fp32: of the two keys (one per half) that score register i is.
        constexpr int GROUPS = S::kHalf ? BN / 16 : NS * 16;
        using VFrag = typename std::conditional<S::kHalf, f16x8, float>::type;
        VFrag vf[GROUPS][ND];
        auto read_v = [&](int i) __attribute__((always_inline)) {
            if constexpr (S::kHalf) {
                const int row = 16 * i + 4 * half + (lane & 15) / 4, row2 = row + 8;
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const int piece = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
                    const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4*)(vb + row * S::ROW + (piece ^ S::swz_v(row)) * 16 + (lane & 1) * 8));
                    const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4*)(vb + row2 * S::ROW + (piece ^ S::swz_v(row2)) * 16 + (lane & 1) * 8));
                    vf[i][d] = __builtin_bit_cast(f16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                }
            } else {
                const int row = (i / 16) * 32 + 8 * (i % 16 / 4) + 4 * half + i % 4;
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const int piece = 8 * d + col / 4;
                    vf[i][d] = *reinterpret_cast<const float*>(vb + row * S::ROW + (piece ^ S::swz_v(row)) * 16 + (col % 4) * 4);
                }
            }
        };
        read_v(0);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MASKED) {
            const int room = limit - k0 - 4 * half;
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool see = n * 32 + 8 * (r / 4) + r % 4 <= room && (valid >> (n * 2 + r / 8) & 1u);
                    s[n][r] = see ? s[n][r] : -INFINITY;
                }
        }
        float bm = s[0][0];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) bm = fmaxf(bm, s[n][r]);
        bm = other_half_max(bm);
        // What the weights are taken against only follows the maximum when that has grown by 2^8 or more: weights of up to 256 lose
        // nothing (a rounding is relative), and a row's sum and output are rescaled a few times, not every few steps.
        if (__builtin_amdgcn_ballot_w64(bm - mx > slack) != 0) {
            const float mnew = bm - mx > slack ? bm : mx;     // (each row by itself: what it gets does not hang on its neighbours)
            const float alpha = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mx - mnew) * a.score_scale);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
            mx = mnew;
            far = __builtin_amdgcn_ballot_w64(is_far(mx)) != 0;
        }
        // fp16 weights are taken times 2^7, the most that leaves room for those 256: ones of 2^-25 or less of the largest - many rows behind
        // one that stands out - would else be lost from the output, not from the sum.
        constexpr float LIFT = S::kHalf ? 7.f : 0.f;
        const float base = mx == -INFINITY ? 0.f : mx;                     // (-inf: a row that has seen nothing yet)
        float shift = base * a.score_scale - LIFT;
        // Far from zero the product of base and scale is rounded by more than a weight can bear (at 2^12 by 2^-13, at 2^25 by 1 - and the
        // weights have 2^0.99 left), so there the scores' differences come first, which are exact where they count.  (8192 tokens: in every
        // step 590 us, behind this branch 577, without it 574)
        if (__builtin_expect(far, 0)) {
            const float own = is_far(mx) ? mx : 0.f;
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[n][r] -= own;
            shift = is_far(mx) ? -LIFT : shift;
        }
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], a.score_scale, -shift));
                l += s[n][r];
            }
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            if (i + 1 < GROUPS) read_v(i + 1);
            if constexpr (S::kHalf) {
                f16x8 pf;
#pragma unroll
                for (int e = 0; e < 8; ++e) pf[e] = (_Float16)s[i / 2][8 * (i % 2) + e];
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[i][d], pf, o[d], 0, 0, 0);
            } else {
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[i][d], s[i / 16][i % 16], o[d], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if (k_begin < k_end) {
        // Steps that every row of the tile sees whole, and whose pages all exist, go in pairs (a buffer pair each) with nothing
        // conditional in between; the rest - the diagonal, as a rule - are masked.
        const int steps = (k_end - k_begin + BN - 1) / BN;
        const int plain = max(0, min(k_end, rows_all) - k_begin) / BN;
        constexpr unsigned kAll = (1u << S::NG) - 1u, kPair = (1u << 2 * S::NG) - 1u;
        auto there_from = [&](int step) __attribute__((always_inline)) { return (unsigned)(there >> (step * S::NG % kWave)); };
        auto arrive = [&]() __attribute__((always_inline)) {               // this wave's rows are there; then everybody's
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        };
        int it = 0, k0 = k_begin, page = 0;
        // (rows behind the last step are requested like the others: their windows are empty)
        auto next = [&](char* kn, char* vn, auto edge_tag) __attribute__((always_inline)) {
            const int step = it + 1;
            if (step % SPB == 0) open_block(step / SPB, page);
            page = pages_of(step / SPB + 1);        // the next block's: asked for in every step, a branch more costs more
            request(kn, vn, step, edge_tag);
        };
        auto plain_step = [&](char* kb, char* vb, char* kn, char* vn, auto edge_tag) __attribute__((always_inline)) {
            next(kn, vn, edge_tag);
            compute(kb, vb, k0, std::false_type{}, kAll);
            arrive();
            ++it;
            k0 += BN;
        };
        auto masked_step = [&](char* kb, char* vb, char* kn, char* vn) __attribute__((always_inline)) {
            const unsigned now = there_from(it) & kAll;
            clean(vb);
            __syncthreads();
            next(kn, vn, std::true_type{});
            compute(kb, vb, k0, std::true_type{}, now);
            arrive();
            ++it;
            k0 += BN;
        };
        open_block(0, pages_of(0));
        request(k_even, v_even, 0, std::true_type{});
        arrive();
        while (it + 2 <= plain && (there_from(it) & kPair) == kPair) {      // (a pair lies in one block)
            plain_step(k_even, v_even, k_odd, v_odd, std::false_type{});
            plain_step(k_odd, v_odd, k_even, v_even, std::true_type{});
        }
        odd_from = k0;                                                   // first key of the masked steps
        while (it < steps) {
            masked_step(k_even, v_even, k_odd, v_odd);
            if (it >= steps) break;
            masked_step(k_odd, v_odd, k_even, v_even);
        }
    }

    l += __shfl_xor(l, 32, kWave);
    // (rare) NaNs and infinities in V.  A weight of any size times such a value is that value - also one that has become zero in the type, whose
    // product with it is NaN - so a component of a row is the sum of those that it sees in the component's column, if there are any.
    // Masked steps left them out (s_odd); plain steps show them by a sum that is not finite although the weights' is.
    bool anywhere = false;
    if (odd_from > k_begin) {
        f32x4 probe = {0.f, 0.f, 0.f, 0.f};                    // (sums of zeros or NaNs)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) probe[r % 4] = __builtin_fmaf(o[d][r], 0.f, probe[r % 4]);
        anywhere = __builtin_amdgcn_ballot_w64((probe[0] + probe[1]) + (probe[2] + probe[3]) != 0.f && l < INFINITY) != 0;
    }
    if (__builtin_expect(k_begin < k_end && (anywhere || __builtin_amdgcn_readfirstlane(s_odd)), 0)) {
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            f32x16 sum;
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[r] = 0.f;
#pragma unroll 1
            for (int row0 = anywhere ? k_begin : odd_from; row0 < k_end; row0 += kRowGroup) {
                const int page = __builtin_amdgcn_readfirstlane(page_of(a.cache, table, row0));
                if (page < 0) continue;
                const T* v = static_cast<const T*>(a.v_pages) + paged_offset(a.cache, page, kvh, row0);
                const __amdgpu_buffer_rsrc_t w = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(v), 0, rows_left(k_end, row0) * D * (int)sizeof(T), 0x00020000);
#pragma unroll 1
                for (int r0 = 0; r0 < kRowGroup; r0 += 4) {           // four rows' loads in flight
                    Quad<T> x[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int r4 = 0; r4 < 4; ++r4) {
                            const int c = 32 * d + 8 * r4 + 4 * half;
                            x[i][r4] = load_quad<T>(w, c < D ? ((r0 + i) * D + c) * (int)sizeof(T) : (int)kOutside);
                        }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const float f = to_f32(x[i][r / 4].v[r % 4]);
                            sum[r] += row0 + r0 + i <= limit && !(__builtin_fabsf(f) < INFINITY) ? f : 0.f;
                        }
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = __builtin_fabsf(sum[r]) < INFINITY ? o[d][r] : sum[r];
        }
    }

    // (rare) No sum although there are rows up to the limit: either none of them has a page, or all scores are -inf, and then there is no
    // distribution - NaN, unless another piece has one: its maximum is above the lowest value that stands here for "saw only -inf".
    bool lost = false;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(l == 0.f && limit >= k_begin) != 0, 0)) {
        for (int block = 0; k_begin + block * kWave * kRowGroup < k_end; ++block) {
            const unsigned long long has = __builtin_amdgcn_ballot_w64(pages_of(block) >= 0);
            const int upto = (limit - k_begin) / kRowGroup - block * kWave;       // the last group of the block that the row sees
            const unsigned long long seen = upto < 0 ? 0 : upto < kWave - 1 ? (2ull << upto) - 1 : ~0ull;
            lost = lost || (l == 0.f && limit >= k_begin && (has & seen) != 0);
        }
        if (lost) mx = kLowest;
    }
    // The sums of a wave go through one of the four buffers, so that whole rows leave it, 16 bytes per lane: as the lanes
    // hold them - 16 bytes each of 32 rows - a row's pieces reach memory apart from each other (four prompts of 1..100 tokens 10.2 us,
    // so 9.7; eight of 1..2048 90.0 and 88.4).
    const bool parts = a.nsplit > 1;
    const float inv = parts ? 1.f : l == 0.f && !lost ? 0.f : 1.f / l;     // (a row that sees no key: zeros)
    const size_t base = (size_t)blockIdx.y * ((size_t)a.token_num * a.Hq);
    if (parts && row_ok && half == 0) {
        const size_t e = base + (size_t)(t.first + token) * a.Hq + head;
        a.part_ml[e * 2] = mx;
        a.part_ml[e * 2 + 1] = l;
    }
    constexpr int COLS = S::TILE / (32 * 4) < DP ? S::TILE / (32 * 4) : DP;     // columns a buffer takes of 32 rows
    __syncthreads();
    float* rows = reinterpret_cast<float*>(wave == 0 ? k_even : wave == 1 ? v_even : wave == 2 ? k_odd : v_odd);
    const int row_left = M - (t.m0 + wave * 32);           // rows of this wave
#pragma unroll
    for (int c0 = 0; c0 < DP; c0 += COLS) {
#pragma unroll
        for (int d = 0; d < COLS / 32; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int piece = 8 * d + 2 * r4 + half;
                const f32x16& x = o[c0 / 32 + d];
                *reinterpret_cast<f32x4*>(rows + col * COLS + (piece ^ (col & 15)) * 4) =
                    f32x4{x[4 * r4] * inv, x[4 * r4 + 1] * inv, x[4 * r4 + 2] * inv, x[4 * r4 + 3] * inv};
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (parts) {
            constexpr int PER = COLS / 4, AT_ONCE = kWave / PER;           // lanes per row; rows at a time
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
                const int r = r0 + lane / PER, piece = lane % PER, c = c0 + piece * 4;
                const f32x4 x = *reinterpret_cast<const f32x4*>(rows + r * COLS + (piece ^ (r & 15)) * 4);
                const int to = __shfl(token, r, kWave), h = __shfl(head, r, kWave);
                if (r < row_left && c < D)
                    // (written through: what the caches still hold when the launch ends is waited for. 512 tokens in two pieces 26.7 us, so 22.3)
                    store16_write_through<false>(a.part_o + (base + (size_t)(t.first + to) * a.Hq + h) * D + c, x);
            }
        } else {
            constexpr int PER = COLS / VEC, AT_ONCE = kWave / PER;
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
                const int r = r0 + lane / PER, piece = lane % PER * (VEC / 4), c = c0 + piece * 4;
                Vec16<T> y;
#pragma unroll
                for (int q = 0; q < VEC / 4; ++q) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(rows + r * COLS + ((piece + q) ^ (r & 15)) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) y.set(4 * q + e, x[e]);
                }
                const int to = __shfl(token, r, kWave), h = __shfl(head, r, kWave);
                if (r < row_left && c < D) store16(static_cast<T*>(a.out) + (size_t)(t.first + to) * a.out_stride + (size_t)h * D + c, y);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1)
void paged_prompt_attn_kernel(const PromptArgs a)
{
    prompt_tile<T, DP>(a);
}

// Joins the pieces of a split call: four columns of one (token, head) per thread, four pieces' states in flight at a time.  Whose
// token it is - one of no sequence has no states and keeps its output - is looked up beside them.
template <typename T>
__global__ __launch_bounds__(256)
void paged_prompt_merge_kernel(const PromptArgs a)
{
    constexpr int BATCH = 4;
    const int nq = a.cache.D / 4;                          // (D is a multiple of four)
    const long rows = (long)a.token_num * a.Hq;
    const int per = 256 / nq;                              // rows of this workgroup
    const int row = (int)blockIdx.x * per + (int)threadIdx.x / nq, c = (int)threadIdx.x % nq * 4;
    if ((int)threadIdx.x >= per * nq || row >= rows) return;
    const int token = row / a.Hq, head = row % a.Hq;
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f}, odd = O;               // (odd: NaNs and infinities, which no weight changes)
    for (int s0 = 0; s0 < a.nsplit; s0 += BATCH) {
        float m[BATCH], l[BATCH];
        f32x4 x[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const long e = min(s0 + j, a.nsplit - 1) * rows + row;
            m[j] = a.part_ml[e * 2];
            l[j] = a.part_ml[e * 2 + 1];
            x[j] = *reinterpret_cast<const f32x4*>(a.part_o + e * a.cache.D + c);
        }
        float bm = M;
#pragma unroll
        for (int j = 0; j < BATCH; ++j) bm = fmaxf(bm, s0 + j < a.nsplit ? m[j] : -INFINITY);
        const float keep = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((M - bm) * a.score_scale);
        L *= keep;
#pragma unroll
        for (int e = 0; e < 4; ++e) O[e] *= keep;
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            // (a piece that saw nothing - no maximum and no sum - has no weight; one whose scores are all NaN has no maximum either, but its sum
            // is NaN, and so is the row)
            const bool on = s0 + j < a.nsplit && (m[j] != -INFINITY || l[j] != 0.f);
            const float w = on ? __builtin_amdgcn_exp2f((m[j] - bm) * a.score_scale) : 0.f;
            L = on ? __builtin_fmaf(l[j], w, L) : L;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool finite = __builtin_fabsf(x[j][e]) < INFINITY;
                O[e] = on && finite ? __builtin_fmaf(x[j][e], w, O[e]) : O[e];
                odd[e] += on && !finite ? x[j][e] : 0.f;
            }
        }
        M = bm;
    }
    int lo = 0, hi = a.B;                                  // the first b with cu[b + 1] > token
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.cu[mid + 1] <= token) lo = mid + 1;
        else hi = mid;
    }
    if (lo >= a.B || token < a.cu[lo] || a.hist[lo] < 0) return;
    const float inv = M == -INFINITY && L == 0.f ? 0.f : 1.f / L;          // (no piece saw a row: zeros; only scores of -inf: 0 / 0)
    T* out = static_cast<T*>(a.out) + (size_t)token * a.out_stride + (size_t)head * a.cache.D + c;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = from_f32<T>((__builtin_fabsf(odd[e]) < INFINITY ? O[e] : odd[e]) * inv);
}

template <typename T>
int launch_prompt(const PromptArgs& a, int tiles, hipStream_t st)
{
    const dim3 grid(a.cache.Hkv, a.nsplit, tiles);
    if (a.cache.D <= 64) hipLaunchKernelGGL((paged_prompt_attn_kernel<T, 64>), grid, dim3(kThreads), 0, st, a);
    else if (a.cache.D <= 128) hipLaunchKernelGGL((paged_prompt_attn_kernel<T, 128>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((paged_prompt_attn_kernel<T, 256>), grid, dim3(kThreads), 0, st, a);
    int rc = launch_status();
    if (rc || a.nsplit == 1) return rc;
    const int rows = a.token_num * a.Hq, per = 256 / (a.cache.D / 4);
    hipLaunchKernelGGL((paged_prompt_merge_kernel<T>), dim3((rows + per - 1) / per), dim3(256), 0, st, a);
    return launch_status();
}

// tiles of all sequences, at most (every sequence may end in a tile of its own)
long tiles_bound(int B, int token_num, int G)
{
    const long rows = (long)token_num * G;
    return rows / kRowsPerTile + (token_num < B ? token_num : B);
}

// Pieces the rows of the cache are cut into.  fp16, 256 workgroups or fewer: the longest tile takes 20 ns per row and 128 columns, so n
// pieces a 1 / n of that (1.45 / n where two share a compute unit, 2 / n with heads above 128, where the second one waits for the
// first); they cost a second launch, 4 us, and each the states' way through memory twice, at 6 TB/s.  The n that is best so, up to two
// workgroups per compute unit and 128 rows per piece.  Heads of 256, 1.45 / 2: 5 tokens of 32 heads on 8 behind 20000 rows 63.0 / 47.9 us, 1000 of
// 8 on 2 behind 3000 76.7 / 63.1, 461 of 16 on 4 behind 15000..20000 247.7 / 246.6; of 160: 61.6 / 46.6, 71.4 / 59.6, 214 / 214.
// 461 tokens behind 15000..20000 rows (120 workgroups) 1 / 2 / 3 / 4 / 5 pieces 404 / 230 / 217 / 185 / 224 us (four), 512 tokens of 32 heads
// on 8 uncut / two 18.1 / 22.3 (uncut), 64 behind 800 uncut / three / six 24.2 / 18.4 / 16.1 (six), 1000 of 8 heads on 2 uncut / three
// 26.4 / 21.1 (three), 1000 of 32 on 8 behind 3000 uncut / two 92.5 / 83.8 (two), 400 behind 1000 two / five 29.5 / 33.1 (two).
// A little more than one workgroup per compute unit, fp16: the longest end long after the others, so two pieces if the tiles' rows
// differ much and are many, as those of one sequence with little before it do, and those of several sequences may - only the device knows
// their lengths, and unequal ones gain more than equal ones lose.  Uncut / two pieces: 4096 tokens of 8
// heads on one (257 workgroups) 88 / 68 us, 6000 (376) 135 / 107, 500 + 500 + 200 tokens behind 500..3000 rows (320) 70 / 59, 8 x 150 behind
// 100..3000 (360) 70 / 60, 4 x 330 behind 6000 each 183 / 177, but 8 x 160 behind 3000 each (384) 96 / 103, 2 x 700 behind 2000 80 / 86; 1400
// tokens (352) 40 / 51, 1100 behind 1000 rows (280) 53 / 65, 1600 behind 6000 (408) 210 / 227.  More workgroups than that are not cut,
// however long one tile is: 5 tokens behind 20000 rows beside 40 prompts of 60 tokens 392 us, in a call of their own 37 and the prompts 20.
// fp32: a tile's steps take six times as long, so the longest tile of a call ends long after the others unless it is cut: three
// workgroups per compute unit (two where heads of more than 128 leave room for one at a time), pieces of 128 rows or more.
// Pieces 1 / 2 / 3 / 4 / 8: 2058 tokens in 4 sequences (264 workgroups) 100 / 85 / 63 / 74 / 87 us, 2048 tokens (520) 384 / 328 / 322 / 345 / 430,
// 1000 (256) 138 / 118 / 115 / 117 / 133, heads of 256: 1024 tokens (136) 288 / 174 / 143 / 142 / 194, 2048 (264) 567 / 360 / 386 / 406 / 546.
int split_of(int dtype, int B, int token_num, long tiles, int Hq, int Hkv, int D, int max_rows)
{
    const long wgs = tiles * Hkv < 1 ? 1 : tiles * Hkv, most = max_rows / 128;
    long n;
    if (dtype != ONELLM_FP16) {
        const long target = D <= 128 ? 768 : 512;
        n = (target + wgs - 1) / wgs;
        if (n > most) n = most;
    } else if (wgs > 256) {
        n = wgs <= 384 && max_rows >= 2048 && (B > 1 || max_rows / 4 * 3 < token_num) ? 2 : 1;
    } else {
        const double whole = max_rows * 0.02 * D / 128.0, piece = 2.0 * token_num * Hq * D * 4.0 / 6e6;      // us
        double best = whole;
        n = 1;
        for (int two = 0; two < 2; ++two) {
            const double sole = two ? (D <= 128 ? 1.45 : 2.0) * whole : whole;
            long c = two ? (512 + wgs / 2) / wgs : 256 / wgs;
            if (c > most) c = most;
            if (c * c * piece > sole) c = (long)(sqrt(sole / piece) + 0.5);
            const double time = sole / c + c * piece + 4.0;
            if (c > 1 && time < best) {
                best = time;
                n = c;
            }
        }
    }
    return n < 1 ? 1 : (int)n;
}

}  // namespace
}  // namespace onellm

extern "C" size_t onellm_paged_prompt_attn_workspace_bytes(int B, int token_num, int Hq, int Hkv, int D, int max_rows)
{
    using namespace onellm;
    if (B <= 0 || token_num <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || max_rows <= 0) return 256;
    const long tiles = tiles_bound(B, token_num, Hq / Hkv);
    const int half = split_of(ONELLM_FP16, B, token_num, tiles, Hq, Hkv, D, max_rows), full = split_of(ONELLM_FP32, B, token_num, tiles, Hq, Hkv, D, max_rows);
    const int n = half > full ? half : full;
    if (n == 1) return 256;
    return (((size_t)n * token_num * Hq * (D + 2) * sizeof(float)) + 255) / 256 * 256;
}

extern "C" int onellm_paged_prompt_attn(int dtype, const void* q, long q_stride, const void* k_pages, const void* v_pages, void* out,
                                        long out_stride, const int* cu_tokens, const int* history_length, const int* block_table,
                                        int B, int token_num, int Hq, int Hkv, int D, int page_size, int num_pages, int max_pages,
                                        int layer, int num_layers, int max_rows, void* workspace, size_t workspace_bytes,
                                        onellm_stream_t stream)
{
    using namespace onellm;
    const int rc = check_paged(dtype, k_pages, v_pages, block_table, B, Hq, Hkv, D, page_size, num_pages, max_pages, layer, num_layers);
    if (rc) return rc;
    if (token_num < 0 || !cu_tokens || !history_length) return ONELLM_EINVAL;
    if (max_rows <= 0) return ONELLM_EINVAL;
    if (token_num == 0) return 0;
    if (!q || !out) return ONELLM_EINVAL;
    const int vec = dtype == ONELLM_FP16 ? 8 : 4;
    if (q_stride < (long)Hq * D || out_stride < (long)Hq * D) return ONELLM_EINVAL;
    if (!aligned16(q) || !aligned16(out) || q_stride % vec != 0 || out_stride % vec != 0) return ONELLM_EUNSUPPORTED;
    const int G = Hq / Hkv;
    const long tiles = tiles_bound(B, token_num, G);
    if ((long)token_num * Hq > 0x3FFFFFFFL || tiles > 65535) return ONELLM_EUNSUPPORTED;
    const bool in_place = q == out && (q_stride == out_stride || token_num == 1);
    if (!in_place && rows_overlap(q, q_stride, (long)Hq * D, out, out_stride, (long)Hq * D, token_num, 16 / vec)) return ONELLM_EINVAL;
    PromptArgs a;
    a.q = q;
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.out = out;
    a.cu = cu_tokens;
    a.hist = history_length;
    a.cache = make_paged(block_table, max_pages, num_pages, page_size, Hkv, D, layer);
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.B = B;
    a.token_num = token_num;
    a.Hq = Hq;
    a.G = G;
    a.score_scale = 1.44269504088896340736f / sqrtf((float)D);
    a.nsplit = split_of(dtype, B, token_num, tiles, Hq, Hkv, D, max_rows);
    a.part_o = nullptr;
    a.part_ml = nullptr;
    if (a.nsplit > 1) {
        if (!workspace || workspace_bytes < onellm_paged_prompt_attn_workspace_bytes(B, token_num, Hq, Hkv, D, max_rows)
            || !aligned16(workspace)) return ONELLM_EWORKSPACE;
        a.part_o = static_cast<float*>(workspace);
        a.part_ml = a.part_o + (size_t)a.nsplit * token_num * Hq * D;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == ONELLM_FP16 ? launch_prompt<__half>(a, (int)tiles, st) : launch_prompt<float>(a, (int)tiles, st);
}
