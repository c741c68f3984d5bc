// Decode attention over a paged key-value cache: one new token per sequence - QKV bias, rotary position t - 1, the new k and v
// rows to their page, attention over the sequence's t rows - in one launch, its rows dealt to the workgroups in equal shares.
//
//   out = sum_j softmax_j(q . k[j] / sqrt(D)) v[j]          2 flops per byte and query head: HBM-bound
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
// multiplied, so they enter at 2^-22; fp32 caches multiply fp32 values.
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
template <int DP>
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
        const float f = __builtin_amdgcn_exp2f(snew[g] - base);
        L += f;
#pragma unroll
        for (int e = 0; e < 4; ++e) O[e] = __builtin_fmaf(sv[c + e], f, O[e]);
    }
    return O;
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
    int rb = u.r0 + wave * RW;
    Pages now = fetch_pages(rb);
    issue_k(now, rb);
    issue_v(now, rb);
    Pages next = fetch_pages(rb + S::RPI);

    // ---- the new token: q of the tile's heads, and in the last piece its k and v rows
    const int QKVH = a.Hq + 2 * a.Hkv;
    const T* qkv = static_cast<const T*>(p.qkv) + (size_t)u.b * QKVH * D;
    const T* bias = static_cast<const T*>(p.bias);
    const int pos = u.t - 1;
    for (int i = tid; i < kHeads * (DP / 2); i += kThr) {
        const int g = i / (DP / 2), pr = i % (DP / 2);
        float x0 = 0.f, x1 = 0.f;
        if (g < ng && 2 * pr < D) {
            const int o = (u.kvh * a.G + u.g0 + g) * D + 2 * pr;
            x0 = to_f32(qkv[o]);
            x1 = to_f32(qkv[o + 1]);
            if (bias) {
                x0 += to_f32(bias[o]);
                x1 += to_f32(bias[o + 1]);
            }
            if (2 * pr < a.rotary_dim) {
                float s, c;
                rope_sincos(pos, rt.f[pr], s, c);
                const float y0 = __builtin_fmaf(x0, c, -(x1 * s));
                x1 = __builtin_fmaf(x1, c, x0 * s);
                x0 = y0;
            }
        }
        sq[g * DP + 2 * pr] = x0 * a.qscale;
        sq[g * DP + 2 * pr + 1] = x1 * a.qscale;
    }
    if (u.is_last) {
        const int page = page_of(p.cache, table, pos);
        const bool keep = u.g0 == 0 && page >= 0;
        const size_t at = keep ? paged_offset(p.cache, page, u.kvh, pos) : 0;
        for (int pr = tid; pr < DP / 2; pr += kThr) {
            float x0 = 0.f, x1 = 0.f, y0 = 0.f, y1 = 0.f;
            if (2 * pr < D) {
                const int ok = (a.Hq + u.kvh) * D + 2 * pr, ov = ok + a.Hkv * D;
                x0 = to_f32(qkv[ok]);
                x1 = to_f32(qkv[ok + 1]);
                y0 = to_f32(qkv[ov]);
                y1 = to_f32(qkv[ov + 1]);
                if (bias) {
                    x0 += to_f32(bias[ok]);
                    x1 += to_f32(bias[ok + 1]);
                    y0 += to_f32(bias[ov]);
                    y1 += to_f32(bias[ov + 1]);
                }
                if (2 * pr < a.rotary_dim) {
                    float s, c;
                    rope_sincos(pos, rt.f[pr], s, c);
                    const float z0 = __builtin_fmaf(x0, c, -(x1 * s));
                    x1 = __builtin_fmaf(x1, c, x0 * s);
                    x0 = z0;
                }
                const T k0 = from_f32<T>(x0), k1 = from_f32<T>(x1), v0 = from_f32<T>(y0), v1 = from_f32<T>(y1);
                if (keep) {
                    T* kd = static_cast<T*>(p.k_pages) + at + 2 * pr;
                    T* vd = static_cast<T*>(p.v_pages) + at + 2 * pr;
                    kd[0] = k0;
                    kd[1] = k1;
                    vd[0] = v0;
                    vd[1] = v1;
                }
                x0 = to_f32(k0);                              // the row as the cache holds it
                x1 = to_f32(k1);
                y0 = to_f32(v0);
                y1 = to_f32(v1);
            }
            sk[2 * pr] = x0;
            sk[2 * pr + 1] = x1;
            sv[2 * pr] = y0;
            sv[2 * pr + 1] = y1;
        }
    }
    __syncthreads();
    if (u.is_last) {
        for (int g = wave; g < kHeads; g += kWaves) {
            float part = 0.f;
            for (int d = lane; d < DP; d += kWave) part = __builtin_fmaf(sq[g * DP + d], sk[d], part);
            part = wave_sum(part);
            if (lane == 0) snew[g] = part;
        }
    }

    // B operand of the scores: column `slot` is head slot, the k slots the columns the K registers hold
    using QFrag = typename std::conditional<S::kHalf, f16x8, f32x4>::type;
    QFrag qhi[NKJ], qlo[S::kHalf ? NKJ : 1];
#pragma unroll
    for (int j = 0; j < NKJ; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float v = sq[slot * DP + (grp + 4 * j) * VEC + e];
            if constexpr (S::kHalf) {
                qhi[j][e] = (_Float16)v;
                qlo[j][e] = (_Float16)(v - (float)qhi[j][e]);
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
            for (int r = 0; r < 4; ++r) s[n][r] = there && rb + n * 16 + 4 * grp + r < r1 ? s0[r] + s1[r] : -INFINITY;
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
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[n][r] = __builtin_amdgcn_exp2f(s[n][r] - base);
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
    if (u.direct) {
        for (int i = tid; i < ng * nq; i += kThr) {
            const int g = i / nq, c = (i % nq) * 4;
            float M, L;
            f32x4 O = join_waves<DP>(st_ml, scratch, snew, sv, u.is_last, g, c, M, L);
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
        const f32x4 O = join_waves<DP>(st_ml, scratch, snew, sv, u.is_last, g, c, M, L);
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

    // weights of the pieces, a head per wave: 2^(m - M) / L
    float* wgt = scratch;                                     // [P][ng]
    for (int g = wave; g < ng; g += kWaves) {
        float M = -INFINITY;
        for (int s = lane; s < P; s += kWave) {
            const auto ml = __builtin_amdgcn_raw_buffer_load_b64(wm, entry(i0 + s, g) * 8u, 0, kDevice);
            M = fmaxf(M, __uint_as_float(ml[0]));
        }
#pragma unroll
        for (int x = 32; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, kWave));
        float L = 0.f;
        for (int s = lane; s < P; s += kWave) {
            const auto ml = __builtin_amdgcn_raw_buffer_load_b64(wm, entry(i0 + s, g) * 8u, 0, kDevice);
            L += __uint_as_float(ml[1]) * __builtin_amdgcn_exp2f(__uint_as_float(ml[0]) - M);
        }
        L = wave_sum(L);
        for (int s = lane; s < P; s += kWave) {
            const auto ml = __builtin_amdgcn_raw_buffer_load_b64(wm, entry(i0 + s, g) * 8u, 0, kDevice);
            wgt[s * ng + g] = __builtin_amdgcn_exp2f(__uint_as_float(ml[0]) - M) / L;
        }
    }
    __syncthreads();
    for (int i = tid; i < ng * nq; i += kThr) {
        const int g = i / nq, c = (i % nq) * 4;
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
        constexpr int BATCH = 8;
        for (int s0 = 0; s0 < P; s0 += BATCH) {
            u32x4 x[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                x[j] = __builtin_amdgcn_raw_buffer_load_b128(wo, (entry(i0 + min(s0 + j, P - 1), g) * D + c) * 4u, 0, kDevice);
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const float f = s0 + j < P ? wgt[min(s0 + j, P - 1) * ng + g] : 0.f;
                const f32x4 y = __builtin_bit_cast(f32x4, x[j]);
#pragma unroll
                for (int e = 0; e < 4; ++e) O[e] = s0 + j < P ? __builtin_fmaf(y[e], f, O[e]) : O[e];
            }
        }
        store_quad<T>(out + (size_t)g * D + c, O);
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
    a.bal_nwg = kBalancedWorkgroups;
    a.unit_cost = 3;
    // item numbers times workgroups have to stay below 2^31 (attn_schedule.hpp)
    while (units * ((longest - 1 + a.item_rows - 1) / a.item_rows + 1 + a.unit_cost) * a.bal_nwg > (long long)kBalancedMaxItemsTimesWorkgroups) {
        if (a.item_rows >= 1 << 20) return ONELLM_EUNSUPPORTED;
        a.item_rows *= 2;
    }
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
