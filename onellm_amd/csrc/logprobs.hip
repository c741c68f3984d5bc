// Log-probabilities of given tokens, entropy and the K likeliest tokens of rows of logits.
//
//   lse = log sum_v exp(x_v);   logprob = x_target - lse;   entropy = lse - sum_v p_v x_v,  p_v = exp(x_v - lse)
//
// One pass: N * V * e bytes read once.  Sums are taken in units of log 2 against a running maximum per thread and joined at
// the end; with y = (x - reference) * log2(e):  Z = sum 2^y,  S = sum 2^y y,  logprob = (x_target - reference) - ln 2 log2 Z,
// entropy = ln 2 (log2 Z - S / Z) - differences only, so a row of large or very negative logits loses nothing.
// Per logit that is a multiply-add, an exponential (two issue slots), an add and for the entropy a clamp and a multiply-add; with
// half a slot for the maximum that is 6.5 slots, 22 us for 4096 x 32000 logits on all SIMDs against 37 us to read them in fp16.  Counted
// are 12.6 slots, 41 us: as much again as the logits' own goes into each row's tail (floor, candidates, joins of 256 lanes), with
// nothing of the next row on its way.
// Measured: 54 us with entropy and the 8 best (46 without the list), 4.8 TB/s; 16 x 32000 fp32 and the 5 best 9.5 us, two launches.
//
// The K best: a wave keeps candidates in LDS as 64-bit keys (value, then lower token first).  The K-th largest of the first step's
// 256 lane maxima, found bit by bit with ballots, is a floor below which nothing can be among the K best; the lanes that reach
// it are looked through, their candidates appended, and the list cut back to the K best, which raises the floor.  Ties and sorted rows only make the list be cut back more often.
//
// Few rows are cut into parts, a workgroup each, and joined by a second launch.
#include "common.hpp"

namespace onellm {
namespace {

typedef unsigned long long Key;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThr = 256, kWaves = kThr / kWave;
constexpr int kPieces = 8;                     // 16-byte pieces per thread and step
constexpr int kMaxK = 32;
constexpr int kList = 256;                     // candidates a wave keeps
constexpr int kStage = 16;                     // lanes whose logits are looked through together
constexpr int kMaxParts = 16;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr unsigned kNegInfKey = 0x007FFFFFu;   // the key word of -inf
constexpr unsigned kOutside = 0x7FFFFF00u;

struct LogprobArgs {
    const void* logits;
    const int* targets;
    float* logprob;
    float* entropy;
    int* top_ids;
    float* top_logprobs;
    long ld;
    int N, V, K;
    int parts, part_len;   // workgroups per row; tokens per part, a multiple of a step (the last part takes the rest)
    float* part_stats;     // [N, parts, 4]: reference, Z, S
    Key* part_keys;        // [N, parts, K]
};

__device__ __forceinline__ unsigned order_of(float v)
{
    const unsigned u = __float_as_uint(v + 0.0f);             // -0 -> +0
    return u ^ ((u & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned o)
{
    return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ Key make_key(float v, int id) { return ((Key)order_of(v) << 32) | (Key)(0xFFFFFFFFu - (unsigned)id); }
__device__ __forceinline__ int id_of(Key k) { return (int)(0xFFFFFFFFu - (unsigned)k); }

// What the sums are taken against.  fp16 logits: in units of log 2, so a logit enters with one multiply-add (its rounding is common to
// the row and cancels).  fp32 logits: the maximum itself - a row masked with the type's lowest value would overflow in units of log 2.
template <typename T> __device__ __forceinline__ float reference_of(float max) { return sizeof(T) == 2 ? max * kLog2e : max; }
template <typename T> __device__ __forceinline__ float exponent(float x, float ref)
{
    return sizeof(T) == 2 ? __builtin_fmaf(x, kLog2e, -ref) : (x - ref) * kLog2e;
}
// What a row's results are made of: its largest logit and log2 of the sum against that.  Of an fp16 row the logit comes back out of the
// reference (its product with log2(e), rounded once: the nearest fp16 value is the logit), and the reference's rounding, which the
// sums carry, is taken off; so a log-probability is a difference of logits and a small logarithm, rounded once, in both types.
struct RowSum { float max, logz; };
template <typename T> __device__ __forceinline__ RowSum row_sum(float ref, float logz)
{
    if constexpr (sizeof(T) == 4) return {ref, logz};
    const float max = (float)(_Float16)(ref * kLn2);
    return {max, logz - __builtin_fmaf(max, kLog2e, -ref)};
}
__device__ __forceinline__ float logprob_of(float x, RowSum r) { return (x - r.max) - r.logz * kLn2; }
template <typename T> __device__ __forceinline__ float exponent_between(float ref, float to)      // of one reference against another
{
    return sizeof(T) == 2 ? ref - to : (ref - to) * kLog2e;
}

struct Stats { float ref, z, s; };             // ref = -inf: nothing but -inf so far

// the sums of `a` and `b` against the larger reference
template <typename T>
__device__ __forceinline__ Stats join(Stats a, Stats b)
{
    Stats r;
    r.ref = fmaxf(a.ref, b.ref);
    const float ea = a.ref == r.ref ? 0.f : fmaxf(exponent_between<T>(a.ref, r.ref), -1e4f);
    const float eb = b.ref == r.ref ? 0.f : fmaxf(exponent_between<T>(b.ref, r.ref), -1e4f);
    const float fa = __builtin_amdgcn_exp2f(ea), fb = __builtin_amdgcn_exp2f(eb);
    r.z = a.z * fa + b.z * fb;
    r.s = fa * __builtin_fmaf(ea, a.z, a.s) + fb * __builtin_fmaf(eb, b.z, b.s);
    return r;
}
template <typename T>
__device__ __forceinline__ Stats join_wave(Stats a)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        Stats b;
        b.ref = __shfl_xor(a.ref, o, kWave);
        b.z = __shfl_xor(a.z, o, kWave);
        b.s = __shfl_xor(a.s, o, kWave);
        a = join<T>(a, b);
    }
    return a;
}

// Cuts a list of n <= 64 * PER keys, all different, to its k best, in order.  Called by one whole wave.  Up to 64 keys are ranked
// out of registers, every key read out of its lane and compared in all of them.  Of a longer list first the keys below the k-th largest
// value are dropped, that value found bit by bit; if ties leave more than 64, the list is ranked against itself in LDS.
__device__ __forceinline__ int rank_list(Key* list, int n, int k)
{
    const int lane = threadIdx.x & (kWave - 1);
    const Key own = lane < n ? list[lane] : 0;
    int rank = 0;
    for (int i0 = 0; i0 < n; i0 += 8) {                       // (keys behind the list are 0, above nothing)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const Key x = (Key)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(own >> 32), i0 + i) << 32
                          | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)own, i0 + i);
            rank += x > own ? 1 : 0;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lane < n && rank < k) list[rank] = own;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return min(n, k);
}

template <int PER>
__device__ __forceinline__ int cut_list(Key* list, int n, int k)
{
    if (n <= kWave) return rank_list(list, n, k);
    const int lane = threadIdx.x & (kWave - 1);
    Key own[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) own[j] = lane + j * kWave < n ? list[lane + j * kWave] : 0;
    unsigned t = 0;                                           // the k-th largest value (k <= 32 < n)
    for (unsigned bit = 0x80000000u; bit; bit >>= 1) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) c += __builtin_popcountll(__builtin_amdgcn_ballot_w64((unsigned)(own[j] >> 32) >= (t | bit)));
        if (c >= k) t |= bit;
    }
    int left = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) left += __builtin_popcountll(__builtin_amdgcn_ballot_w64((unsigned)(own[j] >> 32) >= t));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (left <= kWave) {
        int at = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const bool on = (unsigned)(own[j] >> 32) >= t;
            const unsigned long long who = __builtin_amdgcn_ballot_w64(on);
            if (on) list[at + __builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)who, 0u))] = own[j];
            at += __builtin_popcountll(who);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        return rank_list(list, left, k);
    }
    int rank[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) rank[j] = 0;
    for (int i = 0; i < n; ++i) {
        const Key x = list[i];
#pragma unroll
        for (int j = 0; j < PER; ++j) rank[j] += x > own[j] ? 1 : 0;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (lane + j * kWave < n && rank[j] < k) list[rank[j]] = own[j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return min(n, k);
}

template <typename T>
__device__ __forceinline__ void write_row(const LogprobArgs& a, int row, Stats st, const Key* top, int ntop, int lane)
{
    const T* x = static_cast<const T*>(a.logits) + (size_t)row * a.ld;
    const float logz = __builtin_amdgcn_logf(st.z);           // log2
    const RowSum sum = row_sum<T>(st.ref, logz);
    const bool empty = st.ref == -INFINITY && st.z == 0.f;    // no logit above -inf (and no NaN): no distribution
    if (lane == 0) {
        if (a.logprob) {
            const int t = a.targets[row];
            float v = 0.f;
            if ((unsigned)t < (unsigned)a.V) v = empty ? -INFINITY : logprob_of(to_f32(x[t]), sum);
            a.logprob[row] = v;
        }
        if (a.entropy) a.entropy[row] = empty ? 0.f : (logz - st.s / st.z) * kLn2;
    }
    for (int i = lane; i < a.K; i += kWave) {
        int id = -1;
        float v = -INFINITY;
        if (i < ntop) {
            id = id_of(top[i]);
            v = logprob_of(value_of((unsigned)(top[i] >> 32)), sum);
        }
        a.top_ids[(size_t)row * a.K + i] = id;
        a.top_logprobs[(size_t)row * a.K + i] = v;
    }
}

template <typename T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(kThr)
void token_logprobs_kernel(const LogprobArgs a)
{
    constexpr int VEC = Elt<T>::kVec;
    __shared__ Key lists[TOP ? kWaves : 1][TOP ? kList : 1];
    __shared__ __align__(16) char stage[TOP ? kWaves : 1][TOP ? kStage : 1][kPieces * 16 + 16];
    __shared__ float lane_max[TOP ? kWaves : 1][TOP ? kWave : 1];
    __shared__ int counts[kWaves];
    __shared__ Stats stats[kWaves];
    const int row = blockIdx.x, part = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const T* x = static_cast<const T*>(a.logits) + (size_t)row * a.ld;
    // 16-byte pieces are taken from the aligned address at or before the row's first logit; a piece that is not wholly
    // inside the part is read logit by logit
    const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    const int first = part * a.part_len - skew;               // first logit of the part's first piece
    const int begin = max(first, 0), end = part == a.parts - 1 ? a.V : first + a.part_len;     // logits of the part
    const __amdgpu_buffer_rsrc_t rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(x - skew), 0, (unsigned)((a.V + skew) * (long)sizeof(T)), 0x00020000);

    Stats st{-INFINITY, 0.f, 0.f};
    Key* list = lists[wave];
    int count = 0;
    float floor_v = -INFINITY;                // candidates: above it, or equal to it with a token of floor_id or lower
    int floor_id = 0x7FFFFFFF;
    bool have_floor = false;

    for (int c0 = first; c0 < end; c0 += kThr * kPieces * VEC) {
        Vec16<T> v[kPieces];
        const bool inner = c0 >= begin && c0 + kThr * kPieces * VEC <= end;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int at = c0 + (i * kThr + tid) * VEC;
            const unsigned off = inner || (at >= begin && at + VEC <= end) ? (unsigned)((at + skew) * (int)sizeof(T)) : kOutside;
            v[i].raw = __builtin_bit_cast(decltype(v[i].raw), __builtin_amdgcn_raw_buffer_load_b128(rows, off, 0, 2));
        }
        if (!inner) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int at = c0 + (i * kThr + tid) * VEC;
                if (!(at >= begin && at + VEC <= end)) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        float f = -INFINITY;
                        if (at + e >= begin && at + e < end) f = to_f32(x[at + e]);
                        v[i].set(e, f);
                    }
                }
            }
        }
        float lm = -INFINITY;                 // the lane's maximum
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if constexpr (sizeof(T) == 2) {
                f16x2 h = __builtin_shufflevector(v[i].raw, v[i].raw, 0, 1);
                h = __builtin_elementwise_max(h, __builtin_shufflevector(v[i].raw, v[i].raw, 2, 3));
                h = __builtin_elementwise_max(h, __builtin_shufflevector(v[i].raw, v[i].raw, 4, 5));
                h = __builtin_elementwise_max(h, __builtin_shufflevector(v[i].raw, v[i].raw, 6, 7));
                lm = fmaxf(lm, fmaxf((float)h[0], (float)h[1]));
            } else {
                lm = fmaxf(lm, fmaxf(fmaxf(v[i].get(0), v[i].get(1)), fmaxf(v[i].get(2), v[i].get(3))));
            }
        }
        const float ref = fmaxf(st.ref, reference_of<T>(lm));
        const float old = st.ref == ref ? 0.f : fmaxf(exponent_between<T>(st.ref, ref), -1e4f);
        const float f = __builtin_amdgcn_exp2f(old);
        if (ENTROPY) st.s = f * __builtin_fmaf(old, st.z, st.s);
        st.z *= f;
        st.ref = ref;
        const float base = ref == -INFINITY ? 0.f : ref;      // (only -inf so far: exponents of -inf)
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float y = exponent<T>(v[i].get(e), base);
                const float p = __builtin_amdgcn_exp2f(y);
                st.z += p;
                if (ENTROPY) st.s = __builtin_fmaf(p, fmaxf(y, -1e4f), st.s);       // (0 * -inf)
            }
        if constexpr (TOP) {
            if (!have_floor) {
                // the K-th largest of the workgroup's lane maxima, its 18 leading bits (every wave works it out for itself)
                lane_max[wave][lane] = lm;
                __syncthreads();
                unsigned o[kWaves];
#pragma unroll
                for (int w = 0; w < kWaves; ++w) o[w] = order_of(lane_max[w][lane]);
                unsigned t = 0;
                for (unsigned bit = 0x80000000u; bit >= 0x4000u; bit >>= 1) {
                    int n = 0;
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(o[w] >= (t | bit)));
                    if (n >= a.K) t |= bit;
                }
                if (t > kNegInfKey) floor_v = value_of(t);
                have_floor = true;
            }
            // the lanes whose maximum reaches the floor put their logits into LDS, kStage lanes at a time, where the whole wave
            // looks through one lane's (fp32: two lanes') at once
            bool cut = false;
            unsigned long long who = __builtin_amdgcn_ballot_w64(lm >= floor_v && lm > -INFINITY);
            while (who) {
                const int rank = __builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)who, 0u));
                const bool mine = (who >> lane & 1) && rank < kStage;
                const unsigned long long now = __builtin_amdgcn_ballot_w64(mine);
                if (mine) {
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) *reinterpret_cast<decltype(v[i].raw)*>(stage[wave][rank] + i * 16) = v[i].raw;
                    *reinterpret_cast<int*>(stage[wave][rank] + kPieces * 16) = lane;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                const int n = __builtin_popcountll(now);
                constexpr int EL = kPieces * VEC, AT_ONCE = kWave / EL;        // logits of a lane; lanes looked through at once
                for (int at = 0; at < n; at += 4 * AT_ONCE) {               // (four reads in flight)
                    float q[4];
                    int id[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int from = at + u * AT_ONCE + lane / EL, j = lane % EL;
                        const char* s = stage[wave][min(from, n - 1)];
                        q[u] = from < n ? to_f32(reinterpret_cast<const T*>(s)[j]) : -INFINITY;
                        id[u] = c0 + ((j / VEC) * kThr + wave * kWave + *reinterpret_cast<const int*>(s + kPieces * 16)) * VEC + j % VEC;
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const bool is = q[u] > -INFINITY && (q[u] > floor_v || (q[u] == floor_v && id[u] <= floor_id));
                        const unsigned long long hits = __builtin_amdgcn_ballot_w64(is);
                        if (hits == 0) continue;
                        if (count + __builtin_popcountll(hits) > kList) {
                            count = cut_list<kList / kWave>(list, count, a.K);
                            if (count == a.K) {
                                floor_v = value_of((unsigned)(list[a.K - 1] >> 32));
                                floor_id = id_of(list[a.K - 1]);
                            }
                        }
                        const int before = __builtin_amdgcn_mbcnt_hi((unsigned)(hits >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)hits, 0u));
                        if (is) list[count + before] = make_key(q[u], id[u]);
                        count += __builtin_popcountll(hits);
                        cut = true;
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                who &= ~now;
                who &= __builtin_amdgcn_ballot_w64(lm >= floor_v);             // (a cut may have raised it)
            }
            // (a list of up to 64 is cut once, behind the last step: a floor that is a little low costs less than the cut)
            if (cut && count > kWave) {
                count = cut_list<kList / kWave>(list, count, a.K);
                if (count == a.K) {
                    floor_v = value_of((unsigned)(list[a.K - 1] >> 32));
                    floor_id = id_of(list[a.K - 1]);
                }
            }
        }
    }

    if constexpr (TOP) count = rank_list(list, count, a.K);       // (64 keys at most)
    st = join_wave<T>(st);
    if (lane == 0) {
        stats[wave] = st;
        counts[wave] = count;
    }
    __syncthreads();
    if (wave != 0) return;
    st = stats[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) st = join<T>(st, stats[w]);
    int n = 0;
    if constexpr (TOP) {
        // the waves' lists side by side behind the first one's
        n = counts[0];
        for (int w = 1; w < kWaves; ++w) {
            if (lane < counts[w]) lists[0][n + lane] = lists[w][lane];
            n += counts[w];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        n = cut_list<kWaves * kMaxK / kWave>(lists[0], n, a.K);
    }
    if (a.parts == 1) {
        write_row<T>(a, row, st, lists[0], n, lane);
        return;
    }
    const size_t slot = (size_t)row * a.parts + part;
    if (lane == 0) {
        a.part_stats[slot * 4] = st.ref;
        a.part_stats[slot * 4 + 1] = st.z;
        a.part_stats[slot * 4 + 2] = st.s;
    }
    if (TOP && lane < a.K) a.part_keys[slot * a.K + lane] = lane < n ? lists[0][lane] : 0;
}

// joins the parts of a row: one wave per row
template <typename T>
__global__ __launch_bounds__(kWave)
void token_logprobs_join_kernel(const LogprobArgs a)
{
    __shared__ Key list[kMaxParts * kMaxK];
    const int row = blockIdx.x, lane = threadIdx.x;
    Stats st{-INFINITY, 0.f, 0.f};
    if (lane < a.parts) {
        const float* p = a.part_stats + ((size_t)row * a.parts + lane) * 4;
        st = Stats{p[0], p[1], p[2]};
    }
    int n = 0;
    for (int i0 = 0; i0 < a.parts * a.K; i0 += kWave) {
        const Key k = i0 + lane < a.parts * a.K ? a.part_keys[(size_t)row * a.parts * a.K + i0 + lane] : 0;
        const unsigned long long who = __builtin_amdgcn_ballot_w64(k != 0);
        if (k != 0) list[n + __builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)who, 0u))] = k;
        n += __builtin_popcountll(who);
    }
    st = join_wave<T>(st);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (a.K) n = cut_list<kMaxParts * kMaxK / kWave>(list, n, a.K);
    write_row<T>(a, row, st, list, n, lane);
}

// Parts per row: one where the rows alone give every compute unit two workgroups, else as many as that takes, but at most kMaxParts and
// one per step (16384 logits in fp16, 8192 in fp32), so few rows do not fill the chip.  Whole / in parts: 16 x 32000 fp16, K = 8 (two parts)
// 12.0 / 11.7 us, fp32, K = 5 (four) 13.6 / 11.1; 64 x 128000 fp16 (eight) 30.3 / 14.9; one row of 150000 (ten) 26.1 / 16.9; 300 x 32000 (two)
// 14.4 / 15.3.
int parts_of(int N, int V, int step)
{
    int n = N >= 512 ? 1 : (511 + N) / N;
    const int most = (V + step - 1) / step;
    if (n > most) n = most;
    return n < 1 ? 1 : (n > kMaxParts ? kMaxParts : n);
}

template <typename T>
int launch_logprobs(const LogprobArgs& a, hipStream_t st)
{
    const dim3 grid(a.N, a.parts);
    const bool ent = a.entropy != nullptr, top = a.K > 0;
    if (ent && top) hipLaunchKernelGGL((token_logprobs_kernel<T, true, true>), grid, dim3(kThr), 0, st, a);
    else if (ent) hipLaunchKernelGGL((token_logprobs_kernel<T, true, false>), grid, dim3(kThr), 0, st, a);
    else if (top) hipLaunchKernelGGL((token_logprobs_kernel<T, false, true>), grid, dim3(kThr), 0, st, a);
    else hipLaunchKernelGGL((token_logprobs_kernel<T, false, false>), grid, dim3(kThr), 0, st, a);
    const int rc = launch_status();
    if (rc || a.parts == 1) return rc;
    hipLaunchKernelGGL((token_logprobs_join_kernel<T>), dim3(a.N), dim3(kWave), 0, st, a);
    return launch_status();
}

}  // namespace
}  // namespace onellm

extern "C" size_t onellm_token_logprobs_workspace_bytes(int N, int V, int K)
{
    using namespace onellm;
    if (N <= 0 || V <= 0 || K < 0 || K > kMaxK) return 256;
    // (the finer steps of fp32 rows: at least as many parts as fp16 rows take)
    const size_t parts = parts_of(N, V, kThr * kPieces * 4);
    if (parts == 1) return 256;
    return ((size_t)N * parts * (4 * sizeof(float) + K * sizeof(Key)) + 255) / 256 * 256;
}

extern "C" int onellm_token_logprobs(int dtype, const void* logits, long ld, const int* targets, int N, int V, int K, float* logprob,
                                     float* entropy, int* top_ids, float* top_logprobs, void* workspace, size_t workspace_bytes,
                                     onellm_stream_t stream)
{
    using namespace onellm;
    if (dtype != ONELLM_FP32 && dtype != ONELLM_FP16) return ONELLM_EINVAL;
    if (N < 0 || V <= 0 || K < 0 || ld < V) return ONELLM_EINVAL;
    if (K > kMaxK) return ONELLM_EUNSUPPORTED;
    if (!logprob && !entropy && K == 0) return ONELLM_EINVAL;
    if (N == 0) return 0;
    if (!logits || (logprob && !targets) || (K > 0 && (!top_ids || !top_logprobs))) return ONELLM_EINVAL;
    const int elt = dtype == ONELLM_FP16 ? 2 : 4;
    if (reinterpret_cast<uintptr_t>(logits) % elt != 0) return ONELLM_EINVAL;
    if (V > (1 << 28) || N > (1 << 23)) return ONELLM_EUNSUPPORTED;
    const int step = kThr * kPieces * (16 / elt);
    LogprobArgs a;
    a.logits = logits;
    a.targets = targets;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    a.ld = ld;
    a.N = N;
    a.V = V;
    a.K = K;
    a.parts = parts_of(N, V, step);
    a.part_len = ((V + a.parts - 1) / a.parts + step - 1) / step * step;
    a.parts = (V + a.part_len - 1) / a.part_len;
    a.part_stats = nullptr;
    a.part_keys = nullptr;
    if (a.parts > 1) {
        if (!workspace || workspace_bytes < onellm_token_logprobs_workspace_bytes(N, V, K) || !aligned16(workspace)) return ONELLM_EWORKSPACE;
        a.part_keys = static_cast<Key*>(workspace);
        a.part_stats = reinterpret_cast<float*>(a.part_keys + (size_t)N * a.parts * K);
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == ONELLM_FP16 ? launch_logprobs<__half>(a, st) : launch_logprobs<float>(a, st);
}
