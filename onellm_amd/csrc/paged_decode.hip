// Decode attention over a paged key-value cache: one new token per sequence - QKV bias, rotary position t - 1, the new k and v
// rows to their page, attention over the sequence's t rows - in one launch, its rows dealt to the workgroups in equal shares.
//
//   out = sum_j softmax_j(q . k[j] / sqrt(D)) v[j]          2 flops per byte and query head: HBM-bound
//
// 16 x 4096 rows of 32 kv heads of 128, fp16: 163 us, 6.6 TB/s, the time of the loads alone; 32 x 1024..8192 rows of 8 heads, 32 query
// heads: 100 us; one sequence of 900 rows: 12 us, a chain of dependent loads.
//
// The rows of the step are cut and dealt by the balanced schedule of attn_schedule.hpp (equal cost per workgroup whatever
// the lengths).  A wave takes 16 or 32 rows per step straight into registers, 16 bytes per lane, through windows of 16 rows each
// lie in one page: rows past the piece's end and rows of a page that is none arrive as zeros and are masked, so no load of
// the loop is conditional.  Both products run on the matrix cores, K and V as loaded:
//   S[16 rows x 16 heads] = K Q^T     A = K: lane (slot, grp) holds row `slot`, pieces grp + 4 j
//   O[16 heads x 16 cols] += P V      A = P: the score registers as they are; B = V: lane (slot, grp) holds rows 4 grp + e,
//                                     columns slot * VEC + c: product c takes column c of every lane's piece
// (up to 16 query heads of a kv head are one tile; fewer leave columns unused, the matrix pipe is far from busy).  K registers are
// requested again as soon as the scores are there, V registers behind the output products: one buffer, always in flight.
// Scores, statistics and sums are fp32.  fp16 caches: q and P are fp32 values split into an fp16 part and an fp16 remainder, both
// multiplied, so they enter at 2^-22; fp32 caches multiply fp32 values.  What fp16's narrow range would take away is scaled into it by
// powers of two: q / 4 cannot overflow, its remainder times 2^11 keeps its bits down to a q of 2^-25 (a small q in front of large keys;
// scaling every head by its own largest component cost 2 us of set-up), weights times 2^14 (those of many rows that are 2^-25 or
// less of the largest would else be lost from the output, not from the sum).
#include <type_traits>
#include "attn_schedule.hpp"
#include "paged.hpp"

namespace onellm {
namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kHeads = 16;                     // query heads per tile
constexpr int kWaves = 4, kThr = kWaves * kWave;
constexpr int kMaxWgs = 512;
constexpr size_t kDecodeCounterBytes = 4096;   // arrival counters: one per workgroup of the schedule
static_assert(kMaxWgs * sizeof(int) <= kDecodeCounterBytes && kMaxWgs >= kBalancedWorkgroups, "a counter per workgroup");

struct DecodeArgs {
    AttnArgs a;            // what the schedule reads: t_dev, B, Hkv, G, S (the longest length), bal_nwg, item_rows, unit_cost
    PagedCache cache;
    const void* qkv;
    const void* bias;
    void* k_pages;
    void* v_pages;
    void* out;
    int heads;             // of a tile: min(G, 16)
    int* counters;
    float* part_o;         // [2 * workgroups, heads, D]
    float* part_ml;        // [2 * workgroups, heads, 2]
};

template <typename T, int DP>
struct DecodeShape {
    static constexpr bool kHalf = sizeof(T) == 2;
    static constexpr int VEC = 16 / sizeof(T);
    static constexpr int NT = kHalf || DP <= 64 ? 2 : 1;    // tiles of 16 rows per wave and step
    static constexpr int RW = NT * 16;
    static constexpr int RPI = kWaves * RW;                 // rows per workgroup and step
    static constexpr float LIFT = kHalf ? 16384.f : 1.f;    // what weights, sums and outputs are scaled by until they are divided
    static constexpr int NKJ = DP / (4 * VEC);              // pieces of a K row per lane
    static constexpr int CG = (DP + 16 * VEC - 1) / (16 * VEC);   // groups of 16 pieces of a V row
    static constexpr int ACC = kWaves * kHeads * DP;        // floats: the waves' sums
    static constexpr int SCRATCH = ACC > kMaxWgs * kHeads ? ACC : kMaxWgs * kHeads;   // ... or a weight per piece and head
};

constexpr int kStream = 2;                     // non-temporal
constexpr int kDevice = 16;                    // device scope (sc1): past this quarter's caches
constexpr unsigned kOutside = 0x7FFFFF00u;     // a byte offset no window of 16 rows reaches

__device__ __forceinline__ __amdgpu_buffer_rsrc_t window(const void* p, unsigned bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}

// Statistics and sums of this workgroup's piece for four consecutive columns of a head, out of the waves' states in LDS and - in
// the piece that owns it - the new token's row.
template <typename S, int DP>
__device__ __forceinline__ f32x4 join_waves(const float* st_ml, const float* acc, const float* snew, const float* sv, bool last, int g, int c,
                                            float& M, float& L)
{
    M = last ? snew[g] : -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, st_ml[(w * kHeads + g) * 2]);
    L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    const float base = M == -INFINITY ? 0.f : M;              // (a piece whose rows have no page)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(st_ml[(w * kHeads + g) * 2] - base);
        L = __builtin_fmaf(st_ml[(w * kHeads + g) * 2 + 1], f, L);
        const f32x4 x = *reinterpret_cast<const f32x4*>(acc + (size_t)(w * kHeads + g) * DP + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) O[e] = __builtin_fmaf(x[e], f, O[e]);
    }
    if (last) {
        const float f = __builtin_amdgcn_exp2f(snew[g] - base) * S::LIFT;
        L += f;
#pragma unroll
        for (int e = 0; e < 4; ++e) O[e] = __builtin_fmaf(sv[c + e], f, O[e]);
    }
    return O;
}

// two neighbouring columns of a row
template <typename T> struct alignas(2 * sizeof(T)) Pair { T a, b; };

__device__ __forceinline__ bool all_finite(f32x4 v)
{
    return __builtin_fabsf(v[0]) + __builtin_fabsf(v[1]) + __builtin_fabsf(v[2]) + __builtin_fabsf(v[3]) < INFINITY;
}
__device__ __forceinline__ float odd_part(float v) { return __builtin_fabsf(v) < INFINITY ? 0.f : v; }     // of NaNs and infinities

// four neighbouring columns out of a window
template <typename T>
__device__ __forceinline__ f32x4 load_quad(__amdgpu_buffer_rsrc_t w, unsigned offset)
{
    f32x4 v;
    if constexpr (sizeof(T) == 2) {
        const f16x4 x = __builtin_bit_cast(f16x4, __builtin_amdgcn_raw_buffer_load_b64(w, offset, 0, 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)x[e];
    } else {
        v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(w, offset, 0, 0));
    }
    return v;
}

template <typename T>
__device__ __forceinline__ void store_quad(T* out, f32x4 v)
{
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = from_f32<T>(v[e]);
}

// One piece of a unit: rows [u.r0, u.r1) of a (sequence, kv head, head tile).  A unit in several pieces spans the workgroups
// i0 .. i1; its piece in workgroup w leaves its state in entry 2 w + (w == i0) - a workgroup starts at most one unit that
// it does not finish, and goes on with at most one - and the piece that arrives last at counter i0 joins them.
template <typename T, int DP>
__device__ __forceinline__ void decode_piece(const DecodeArgs& p, const RopeTurns& rt, Unit u, int i0, int i1, float* lds)
{
    // the same in every lane: said here, behind the walk's divisions and branches, so that all that follows stays scalar
    u.b = uniform(u.b);
    u.kvh = uniform(u.kvh);
    u.g0 = uniform(u.g0);
    u.t = uniform(u.t);
    u.r0 = uniform(u.r0);
    u.r1 = uniform(u.r1);
    using S = DecodeShape<T, DP>;
    constexpr int VEC = S::VEC, NT = S::NT, NKJ = S::NKJ, CG = S::CG, RW = S::RW;
    const AttnArgs& a = p.a;
    const int D = p.cache.D;
    float* sq = lds;                           // [kHeads][DP]
    float* sk = sq + kHeads * DP;              // [DP]
    float* sv = sk + DP;                       // [DP]
    float* snew = sv + DP;                     // [kHeads]
    float* st_ml = snew + kHeads;              // [kWaves][kHeads][2]
    float* scratch = st_ml + kWaves * kHeads * 2;

    const int tid = lane_id_per_unit();
    const int lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int slot = lane & 15, grp = lane >> 4;
    const int ng = min(p.heads, a.G - u.g0);   // heads of this tile
    const int* table = p.cache.table + (size_t)u.b * p.cache.max_pages;
    const int r1 = u.r1;

    // ---- the rows' loads
    unsigned koff[NKJ], voff[CG];              // byte offsets inside a window; pieces behind the head's end lie outside
#pragma unroll
    for (int j = 0; j < NKJ; ++j) {
        const int c = (grp + 4 * j) * VEC;
        koff[j] = c < D ? (unsigned)((slot * D + c) * (int)sizeof(T)) : kOutside;
    }
#pragma unroll
    for (int g = 0; g < CG; ++g) {
        const int c = (g * 16 + slot) * VEC;
        voff[g] = c < D ? (unsigned)((4 * grp * D + c) * (int)sizeof(T)) : kOutside;
    }
    Vec16<T> kr[NT][NKJ], vr[NT][CG][4];
    typedef int Pages __attribute__((ext_vector_type(2)));
    auto fetch_pages = [&](int rb) __attribute__((always_inline)) {       // pages of the wave's rows rb ..
        Pages g = {-1, -1};
        if (rb < r1) g.x = __builtin_amdgcn_readfirstlane(page_of(p.cache, table, rb));
        if (NT > 1 && rb + kRowGroup < r1) g.y = __builtin_amdgcn_readfirstlane(page_of(p.cache, table, rb + kRowGroup));
        return g;
    };
    auto row_window = [&](const void* pages, int page, int row0) __attribute__((always_inline)) {
        const int rows = page < 0 ? 0 : rows_left(r1, row0);
        return window(static_cast<const T*>(pages) + paged_offset(p.cache, max(page, 0), u.kvh, row0), rows * D * (int)sizeof(T));
    };
    auto issue_k = [&](Pages g, int rb) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const __amdgpu_buffer_rsrc_t w = row_window(p.k_pages, n ? g.y : g.x, rb + n * kRowGroup);
#pragma unroll
            for (int j = 0; j < NKJ; ++j)
                kr[n][j].raw = __builtin_bit_cast(decltype(kr[n][j].raw), __builtin_amdgcn_raw_buffer_load_b128(w, koff[j], 0, kStream));
        }
    };
    auto issue_v = [&](Pages g, int rb) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const __amdgpu_buffer_rsrc_t w = row_window(p.v_pages, n ? g.y : g.x, rb + n * kRowGroup);
#pragma unroll
            for (int cg = 0; cg < CG; ++cg)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    vr[n][cg][e].raw = __builtin_bit_cast(decltype(vr[n][cg][e].raw),
                                                          __builtin_amdgcn_raw_buffer_load_b128(w, voff[cg], e * D * (int)sizeof(T), kStream));
        }
    };
    // ---- the new token: q of the tile's heads, and in the last piece its k and v row, a pair of columns per thread at a
    // time, two pairs' loads together.  The first ones set out before the rows' first loads: loads return in order, and the set-up
    // then runs while the rows are on their way (behind them it waited for 64 KiB per compute unit).
    const int QKVH = a.Hq + 2 * a.Hkv;
    const T* qkv = static_cast<const T*>(p.qkv) + (size_t)u.b * QKVH * D;
    const T* bias = static_cast<const T*>(p.bias);
    const int pos = u.t - 1, half_d = D / 2;
    const float qscale = S::kHalf ? a.qscale * 0.25f : a.qscale;
    const int rows_new = ng + (u.is_last ? 2 : 0);            // heads of q, then k, then v
    Pair<T> nx[2], ny[2];
    int ng_[2], npair[2];
    auto request_new = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = min(i0 + j * kThr, rows_new * half_d - 1);
            ng_[j] = i / half_d;
            npair[j] = i - ng_[j] * half_d;
            const int head = ng_[j] < ng ? u.kvh * a.G + u.g0 + ng_[j] : a.Hq + u.kvh + (ng_[j] - ng) * a.Hkv;
            nx[j] = *reinterpret_cast<const Pair<T>*>(qkv + head * D + 2 * npair[j]);
            ny[j] = bias ? *reinterpret_cast<const Pair<T>*>(bias + head * D + 2 * npair[j]) : Pair<T>{};
        }
    };
    request_new(tid);
    asm volatile("" ::: "memory");                            // (the requests stay in front of the rows')

    int rb = u.r0 + wave * RW;
    Pages now = fetch_pages(rb);
    issue_k(now, rb);
    issue_v(now, rb);
    Pages next = fetch_pages(rb + S::RPI);

    const int new_page = u.is_last ? page_of(p.cache, table, pos) : -1;
    const bool keep = u.g0 == 0 && new_page >= 0;
    const size_t new_at = keep ? paged_offset(p.cache, new_page, u.kvh, pos) : 0;
    for (int i0 = tid; i0 < rows_new * half_d; i0 += 2 * kThr) {
        if (i0 != tid) request_new(i0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (i0 + j * kThr >= rows_new * half_d) continue;
            const int g = ng_[j], pr = npair[j];
            float x0 = to_f32(nx[j].a), x1 = to_f32(nx[j].b);
            if (bias) {                                       // (adding zero would turn -0 into +0, which the store does not)
                x0 += to_f32(ny[j].a);
                x1 += to_f32(ny[j].b);
            }
            if (g <= ng && 2 * pr < a.rotary_dim) {
                float sn, cs;
                rope_sincos(pos, rt.f[pr], sn, cs);
                const float r0 = __builtin_fmaf(x0, cs, -(x1 * sn));
                x1 = __builtin_fmaf(x1, cs, x0 * sn);
                x0 = r0;
            }
            if (g < ng) {
                sq[g * DP + 2 * pr] = x0 * qscale;
                sq[g * DP + 2 * pr + 1] = x1 * qscale;
            } else {
                const Pair<T> v{from_f32<T>(x0), from_f32<T>(x1)};
                float* d = g == ng ? sk : sv;                 // the row as the cache holds it
                d[2 * pr] = to_f32(v.a);
                d[2 * pr + 1] = to_f32(v.b);
                if (keep) *reinterpret_cast<Pair<T>*>(static_cast<T*>(g == ng ? p.k_pages : p.v_pages) + new_at + 2 * pr) = v;
            }
        }
    }
    __syncthreads();
    if (u.is_last) {
        for (int g = wave; g < ng; g += kWaves) {
            float part = 0.f;
            for (int d = lane; d < D; d += kWave) part = __builtin_fmaf(sq[g * DP + d], sk[d], part);
            part = wave_sum(part);
            if (lane == 0) snew[g] = S::kHalf ? part * 4.f : part;
        }
    }

    // B operand of the scores: column `slot` is head slot, the k slots the columns the K registers hold
    using QFrag = typename std::conditional<S::kHalf, f16x8, f32x4>::type;
    QFrag qhi[NKJ], qlo[S::kHalf ? NKJ : 1];
#pragma unroll
    for (int j = 0; j < NKJ; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float v = slot < ng && (grp + 4 * j) * VEC < D ? sq[slot * DP + (grp + 4 * j) * VEC + e] : 0.f;
            if constexpr (S::kHalf) {
                qhi[j][e] = (_Float16)v;
                qlo[j][e] = (_Float16)((v - (float)qhi[j][e]) * 2048.f);
            } else {
                qhi[j][e] = v;
            }
        }

    // ---- the rows
    float m = -INFINITY, l = 0.f;              // of head `slot` (m the same in all four grp, l this lane's share)
    f32x4 o[CG][VEC];                          // heads 4 grp + r, column (cg * 16 + slot) * VEC + c
#pragma unroll
    for (int cg = 0; cg < CG; ++cg)
#pragma unroll
        for (int c = 0; c < VEC; ++c) o[cg][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int steps = r1 > u.r0 ? (r1 - u.r0 + S::RPI - 1) / S::RPI : 0;
    for (int it = 0; it < steps; ++it) {
        f32x4 s[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
            for (int j = 0; j < NKJ; ++j) {
                if constexpr (S::kHalf) {
                    s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kr[n][j].raw, qhi[j], s0, 0, 0, 0);
                    s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kr[n][j].raw, qlo[j], s1, 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[n][j].raw[e], qhi[j][e], s0, 0, 0, 0);
                        s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[n][j].raw[e + 1], qhi[j][e + 1], s1, 0, 0, 0);
                    }
                }
            }
            const bool there = (n ? now.y : now.x) >= 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) s[n][r] = there && rb + n * 16 + 4 * grp + r < r1 ? (S::kHalf ? __builtin_fmaf(s0[r], 4.f, s1[r] * (4.f / 2048.f)) : s0[r] + s1[r]) : -INFINITY;
        }
        issue_k(next, rb + S::RPI);
        float bm = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
        if constexpr (NT > 1) bm = fmaxf(bm, fmaxf(fmaxf(s[NT - 1][0], s[NT - 1][1]), fmaxf(s[NT - 1][2], s[NT - 1][3])));
        if (__builtin_amdgcn_ballot_w64(bm > m) != 0) {
            bm = fmaxf(bm, __shfl_xor(bm, 16, kWave));
            bm = fmaxf(bm, __shfl_xor(bm, 32, kWave));
            const float mnew = fmaxf(m, bm);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mnew);
            l *= alpha;
            float al[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) al[r] = __shfl(alpha, (lane & 48) | (4 * grp + r), kWave);
#pragma unroll
            for (int cg = 0; cg < CG; ++cg)
#pragma unroll
                for (int c = 0; c < VEC; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[cg][c][r] *= al[r];
            m = mnew;
        }
        // (the lift is a factor, not part of the exponent: next to a score of 2^25 and more 14 would be rounded to 16, and the largest weights
        // would leave fp16)
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[n][r] = __builtin_amdgcn_exp2f(s[n][r] - base) * S::LIFT;
                l += s[n][r];
            }
        if constexpr (S::kHalf) {
            static_assert(NT == 2, "32 rows per product");
            f16x8 phi, plo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = s[e / 4][e % 4];
                phi[e] = (_Float16)v;
                plo[e] = (_Float16)(v - (float)phi[e]);
            }
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) {
                u32x4 w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = __builtin_bit_cast(u32x4, vr[e / 4][cg][e % 4].raw);
#pragma unroll
                for (int c = 0; c < VEC; ++c) {
                    // column c of the eight rows: one byte-permute per pair of rows
                    const unsigned sel = (c & 1) ? 0x07060302u : 0x05040100u;
                    u32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_perm(w[2 * e + 1][c / 2], w[2 * e][c / 2], sel);
                    const f16x8 vf = __builtin_bit_cast(f16x8, v);
                    o[cg][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(phi, vf, o[cg][c], 0, 0, 0);
                    o[cg][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(plo, vf, o[cg][c], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int cg = 0; cg < CG; ++cg)
#pragma unroll
                        for (int c = 0; c < VEC; ++c)
                            o[cg][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(s[n][r], vr[n][cg][r].raw[c], o[cg][c], 0, 0, 0);
        }
        rb += S::RPI;
        issue_v(next, rb);
        now = next;
        next = fetch_pages(rb + S::RPI);
    }

    // ---- the waves' states meet in LDS
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
    if (grp == 0) {
        st_ml[(wave * kHeads + slot) * 2] = m;
        st_ml[(wave * kHeads + slot) * 2 + 1] = l;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (4 * grp + r < ng) {
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) {
                const int c0 = (cg * 16 + slot) * VEC;
                if (c0 < DP) {
                    float* d = scratch + (size_t)(wave * kHeads + 4 * grp + r) * DP + c0;
#pragma unroll
                    for (int c = 0; c < VEC; c += 4)
                        *reinterpret_cast<f32x4*>(d + c) = f32x4{o[cg][c][r], o[cg][c + 1][r], o[cg][c + 2][r], o[cg][c + 3][r]};
                }
            }
        }
    __syncthreads();
    const int nq = D / 4;                                     // quads of a head
    T* out = static_cast<T*>(p.out) + ((size_t)u.b * a.Hq + u.kvh * a.G + u.g0) * D;
    // (rare) NaNs and infinities in V: a component is the sum of those in its column, whatever their weights.  A weight that is zero in the type, or
    // the remainder of one, makes NaN of an infinity; so where a sum is not finite although the weights' is, the piece's rows are looked
    // through for such values.  (Here and not on the waves' sums: there it waited for the rows requested behind the last step, 0.4 us)
    auto odd_values = [&](f32x4 O, float L, int c) __attribute__((always_inline)) {
        if (__builtin_expect(!all_finite(O) && L < INFINITY, 0)) {
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int row0 = u.r0; row0 < r1; row0 += kRowGroup) {
                const int page = __builtin_amdgcn_readfirstlane(page_of(p.cache, table, row0));
                const __amdgpu_buffer_rsrc_t w = row_window(p.v_pages, page, row0);
#pragma unroll
                for (int r = 0; r < kRowGroup; ++r) {
                    const f32x4 x = load_quad<T>(w, (unsigned)((r * D + c) * (int)sizeof(T)));
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] += odd_part(x[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (u.is_last) sum[e] += odd_part(sv[c + e]);
                O[e] = __builtin_fabsf(sum[e]) < INFINITY ? O[e] : sum[e];
            }
        }
        return O;
    };
    if (u.direct) {
        for (int i = tid; i < ng * nq; i += kThr) {
            const int g = i / nq, c = (i % nq) * 4;
            float M, L;
            f32x4 O = join_waves<S, DP>(st_ml, scratch, snew, sv, u.is_last, g, c, M, L);
            O = odd_values(O, L, c);
            const float inv = 1.f / L;                        // (the new token's row is always there)
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] *= inv;
            store_quad<T>(out + (size_t)g * D + c, O);
        }
        return;
    }

    // ---- a piece of several: publish, arrive, and the last one joins.  What orders the hand-over between chip quarters is
    // what orders the fused finish of the contiguous cache's kernel (attn_finish.hpp, finish_unit): the state goes out with
    // device-scope stores, which drop from vmcnt only when memory has acknowledged them; every wave waits for its own before the
    // barrier, behind which thread 0 adds to the counter, an atomic executed at memory; the piece that finds all others arrived
    // reads their states with device-scope loads, which no cache of its quarter answers.
    const int wg = blockIdx.x, entries = 2 * kMaxWgs;
    const __amdgpu_buffer_rsrc_t wo = window(p.part_o, (unsigned)(entries * p.heads * D * (int)sizeof(float)));
    const __amdgpu_buffer_rsrc_t wm = window(p.part_ml, (unsigned)(entries * p.heads * 2 * (int)sizeof(float)));
    auto entry = [&](int w, int g) __attribute__((always_inline)) { return (unsigned)((2 * w + (w == i0 ? 1 : 0)) * p.heads + g); };
    for (int i = tid; i < ng * nq; i += kThr) {
        const int g = i / nq, c = (i % nq) * 4;
        float M, L;
        f32x4 O = join_waves<S, DP>(st_ml, scratch, snew, sv, u.is_last, g, c, M, L);
        O = odd_values(O, L, c);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, O), wo, (entry(wg, g) * D + c) * 4u, 0, kDevice);
        if (c == 0) {
            typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
            __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(M), __float_as_uint(L)}, wm, entry(wg, g) * 8u, 0, kDevice);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* arrived = reinterpret_cast<int*>(st_ml);
    if (tid == 0) *arrived = __hip_atomic_fetch_add(p.counters + i0, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const int P = i1 - i0 + 1;
    if (*arrived != P - 1) return;
    if (tid == 0) __hip_atomic_store(p.counters + i0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);    // zero for the next call

    // The first batch of sums sets out beside the statistics; their weights - 2^(m - M) / L, a head per wave - are worked out
    // meanwhile.  A thread takes a quad of columns and, where there are fewer quads than threads, every `slices`-th batch of pieces.
    constexpr int BATCH = 4;
    const int quads = ng * nq, slices = max(1, kThr / quads);
    const int quad = tid % quads, slice = tid / quads;
    float* wgt = scratch;                                     // [P][ng]
    f32x4* part = reinterpret_cast<f32x4*>(lds);              // [slices][quads] (q and the new rows are no longer needed)
    const int rounds = (quads + kThr - 1) / kThr;
    for (int round = 0; round < rounds; ++round) {
        const int i = slices > 1 ? quad : tid + round * kThr;
        const bool on = slices > 1 ? slice < slices : i < quads;
        const int g = on ? i / nq : 0, c = on ? (i - g * nq) * 4 : 0;
        const int first = slices > 1 ? slice : 0;
        u32x4 x[BATCH];
        auto fetch = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                x[j] = __builtin_amdgcn_raw_buffer_load_b128(wo, (entry(i0 + min(s0 + j, P - 1), g) * D + c) * 4u, 0, kDevice);
        };
        fetch(first * BATCH);
        if (round == 0) {
            for (int h = wave; h < ng; h += kWaves) {
                float M = -INFINITY, L = 0.f;
                for (int s = lane; s < P; s += kWave) {
                    const auto ml = __builtin_amdgcn_raw_buffer_load_b64(wm, entry(i0 + s, h) * 8u, 0, kDevice);
                    const float pm = __uint_as_float(ml[0]), pl = __uint_as_float(ml[1]);
                    wgt[s * ng + h] = pm;
                    const float top = fmaxf(M, pm);           // (a piece that saw nothing: -inf, and no sum)
                    const float base = top == -INFINITY ? 0.f : top;
                    L = L * __builtin_amdgcn_exp2f(M - base) + pl * __builtin_amdgcn_exp2f(pm - base);
                    M = top;
                }
                float top = M;
#pragma unroll
                for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, kWave));
                L = wave_sum(L * __builtin_amdgcn_exp2f(M - top));           // (the new token's piece has a finite maximum)
                for (int s = lane; s < P; s += kWave) wgt[s * ng + h] = __builtin_amdgcn_exp2f(wgt[s * ng + h] - top) / L;
            }
            __syncthreads();
        }
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = first * BATCH; s0 < P; s0 += slices * BATCH) {
            if (s0 != first * BATCH) fetch(s0);
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const float f = wgt[min(s0 + j, P - 1) * ng + g];
                const f32x4 y = __builtin_bit_cast(f32x4, x[j]);
#pragma unroll
                for (int e = 0; e < 4; ++e) O[e] = s0 + j < P ? __builtin_fmaf(y[e], f, O[e]) : O[e];
            }
        }
        if (__builtin_expect(!all_finite(O), 0)) {            // (rare) the pieces' NaNs and infinities are not weighted
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int s0 = first * BATCH; s0 < P; s0 += slices * BATCH) {
                fetch(s0);
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const float f = wgt[min(s0 + j, P - 1) * ng + g];
                    const f32x4 y = __builtin_bit_cast(f32x4, x[j]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] += s0 + j < P ? __builtin_fmaf(f, 0.f, odd_part(y[e])) : 0.f;       // (a NaN weight wins)
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] = __builtin_fabsf(sum[e]) < INFINITY ? O[e] : sum[e];
        }
        if (slices > 1) {
            if (on) part[slice * quads + quad] = O;
            __syncthreads();
            if (slice == 0) {
                for (int x = 1; x < min(slices, (P + BATCH - 1) / BATCH); ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) O[e] += part[x * quads + quad][e];
                store_quad<T>(out + (size_t)g * D + c, O);
            }
        } else if (on) {
            store_quad<T>(out + (size_t)g * D + c, O);
        }
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(kThr, DP <= 128 ? 2 : 1)
void paged_decode_attn_kernel(const DecodeArgs p, const RopeTurns rt)
{
    using S = DecodeShape<T, DP>;
    __shared__ __align__(16) float lds[kHeads * DP + 2 * DP + kHeads + kWaves * kHeads * 2 + S::SCRATCH];
    const AttnArgs& a = p.a;
    Walk w;
    if (!walk_begin(a, a.Hkv * ((a.G + kHeads - 1) / kHeads), w)) return;
    while (w.cur < w.hi) {
        Unit u;
        int nitems;
        const bool rows = walk_unit<kHeads>(a, w, u, nitems);
        if (rows) {
            int i0 = 0, i1 = 0;
            if (!u.direct) {
                const unsigned first = w.base + (unsigned)(u.counter - w.b * w.nunits) * (unsigned)w.items;
                i0 = uniform(item_owner(first + (unsigned)a.unit_cost, w.W, w.N));
                i1 = uniform(item_owner(first + (unsigned)w.items - 1u, w.W, w.N));
            }
            decode_piece<T, DP>(p, rt, u, i0, i1, lds);
        }
        walk_advance(a, w, nitems);
        if (rows && w.cur < w.hi) __syncthreads();            // the next unit reuses the LDS
    }
}

__global__ void paged_decode_clear_kernel(int* counters)
{
    counters[threadIdx.x] = 0;
}

template <typename T>
void launch_decode(const DecodeArgs& p, const RopeTurns& rt, hipStream_t st)
{
    const dim3 grid(p.a.bal_nwg);
    if (p.cache.D <= 64) hipLaunchKernelGGL((paged_decode_attn_kernel<T, 64>), grid, dim3(kThr), 0, st, p, rt);
    else if (p.cache.D <= 128) hipLaunchKernelGGL((paged_decode_attn_kernel<T, 128>), grid, dim3(kThr), 0, st, p, rt);
    else hipLaunchKernelGGL((paged_decode_attn_kernel<T, 256>), grid, dim3(kThr), 0, st, p, rt);
}

}  // namespace
}  // namespace onellm

extern "C" size_t onellm_paged_decode_attn_workspace_bytes(int B, int Hq, int Hkv, int D, int max_t)
{
    using namespace onellm;
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || D > kPagedMaxD || max_t <= 0) return 256;
    const size_t heads = Hq / Hkv < kHeads ? Hq / Hkv : kHeads;
    return kDecodeCounterBytes + (2 * (size_t)kMaxWgs * heads * (D + 2) * sizeof(float) + 255) / 256 * 256;
}

extern "C" int onellm_paged_decode_attn(int dtype, const void* qkv, const void* qkv_bias, void* k_pages, void* v_pages, void* out,
                                        const int* block_table, const int* t_dev, int B, int Hq, int Hkv, int D, int page_size,
                                        int num_pages, int max_pages, int layer, int num_layers, int max_t, int rotary_dim,
                                        float rope_base, unsigned flags, void* workspace, size_t workspace_bytes, onellm_stream_t stream)
{
    using namespace onellm;
    const int rc = check_paged(dtype, k_pages, v_pages, block_table, B, Hq, Hkv, D, page_size, num_pages, max_pages, layer, num_layers);
    if (rc) return rc;
    if (!qkv || !out || !t_dev || max_t <= 0 || (flags & ~ONELLM_ATTN_ZEROED_WORKSPACE)) return ONELLM_EINVAL;
    if (rotary_dim < 0 || rotary_dim % 2 != 0 || (rotary_dim > 0 && !(rope_base > 0.f && rope_base < INFINITY))) return ONELLM_EINVAL;
    if (!aligned16(qkv) || !aligned16(out) || (qkv_bias && !aligned16(qkv_bias))) return ONELLM_EUNSUPPORTED;
    if (!workspace || !aligned16(workspace) || workspace_bytes < onellm_paged_decode_attn_workspace_bytes(B, Hq, Hkv, D, max_t))
        return ONELLM_EWORKSPACE;
    const long long rows = (long long)page_size * max_pages;
    const int longest = (int)(max_t < rows ? max_t : rows);
    const int G = Hq / Hkv;
    const long long units = (long long)B * Hkv * ((G + kHeads - 1) / kHeads);
    DecodeArgs p{};
    AttnArgs& a = p.a;
    a.t_dev = t_dev;
    a.B = B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.G = G;
    a.S = longest;
    a.rotary_dim = rotary_dim;
    a.qscale = 1.44269504088896340736f / sqrtf((float)D);
    a.item_rows = 64;
    // One share per compute unit, two where there are many short units (a second workgroup then covers the first one's set-up and
    // finish; with long units the two end far apart).  16 sequences x 32 kv heads of 128, fp16, one / two shares: 512 rows
    // 29.0 / 24.6 us, 1024 rows 48.4 / 44.7, 4096 rows 163.4 / 167.6; 96 x 8 heads of 100..1000 rows 54.6 / 50.9; 32 x 8 of
    // 1024..8192 rows 100.1 / 101.4; 8 x 8 of 256..2048 rows 16.2 / 18.9; 32 x 8 heads of 64, 512..4096 rows 39.5 / 38.3.
    // A change of unit costs a workgroup about 1.5 KiB x 64 of each cache's bytes, half that where another workgroup fills in.
    const long long row_bytes = (long long)D * (dtype == ONELLM_FP16 ? 2 : 4);
    const bool two = units >= kBalancedWorkgroups / 2 && longest * row_bytes <= 512 << 10;
    a.bal_nwg = two ? kBalancedWorkgroups : kBalancedWorkgroups / 2;
    a.unit_cost = (int)((two ? 768 : 1536) / row_bytes);
    if (a.unit_cost < 1) a.unit_cost = 1;
    if (a.unit_cost > 12) a.unit_cost = 12;
    // item numbers times workgroups have to stay below 2^31 (attn_schedule.hpp)
    while (units * ((longest - 1 + a.item_rows - 1) / a.item_rows + 1 + a.unit_cost) * a.bal_nwg > (long long)kBalancedMaxItemsTimesWorkgroups) {
        if (a.item_rows >= 1 << 20) return ONELLM_EUNSUPPORTED;
        a.item_rows *= 2;
    }
    if (rows_overlap(qkv, 0, (long)B * (Hq + 2 * Hkv) * D, out, 0, (long)B * Hq * D, 1, (size_t)(row_bytes / D))) return ONELLM_EINVAL;
    p.cache = make_paged(block_table, max_pages, num_pages, page_size, Hkv, D, layer);
    p.qkv = qkv;
    p.bias = qkv_bias;
    p.k_pages = k_pages;
    p.v_pages = v_pages;
    p.out = out;
    p.heads = G < kHeads ? G : kHeads;
    p.counters = static_cast<int*>(workspace);
    p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + kDecodeCounterBytes);
    p.part_ml = p.part_o + 2 * (size_t)kMaxWgs * p.heads * D;
    RopeTurns rt;
    fill_rope_turns(rt, D, rotary_dim, rope_base);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (!(flags & ONELLM_ATTN_ZEROED_WORKSPACE)) {
        hipLaunchKernelGGL(paged_decode_clear_kernel, dim3(1), dim3(kMaxWgs), 0, st, p.counters);
        const int e = launch_status();
        if (e) return e;
    }
    if (dtype == ONELLM_FP16) launch_decode<__half>(p, rt, st);
    else launch_decode<float>(p, rt, st);
    return launch_status();
}
