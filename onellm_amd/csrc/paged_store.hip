// Packed tokens into a paged key-value cache: QKV bias, rotary positions, q to its buffer, k and v rows to their pages.
//
// HBM-bound: every element is read once and written once, 2 * tokens * (Hq + 2 Hkv) * D * e bytes.  4 x 2048 tokens, 96 heads of 128,
// fp16: 75 us, 5.4 TB/s (a plain device copy: 5.15).  4 x 8 tokens of 48 heads: 4 us, a launch and three dependent loads.
#include "paged.hpp"

namespace onellm {
namespace {

struct StoreArgs {
    void* q_out;
    void* k_pages;
    void* v_pages;
    const void* qkv;
    const void* bias;
    const int* cu;
    const int* hist;
    PagedCache cache;
    long q_stride;
    int B, token_num, Hq, rotary_dim;
    int nvec, tokens, heads;   // 16-byte pieces of a row; tokens and heads (per slice) a workgroup takes
};

// A thread keeps one 16-byte piece of one token's rows and walks the heads of its slice: the place of the token - its
// sequence, position, page - and the sines and cosines of the piece's pairs are worked out once, while the first heads' rows are on
// their way.  The lanes of a wave cover the same head of consecutive tokens, which are neighbours in their page.
template <typename T>
__global__ __launch_bounds__(256)
void paged_qkv_store_kernel(const StoreArgs a, const RopeTurns rt)
{
    constexpr int VEC = Elt<T>::kVec, UNROLL = 8;
    const int tid = threadIdx.x;
    const int group = a.nvec * a.tokens;            // threads that share a head
    const int hpp = 256 / group;                    // heads per pass
    const int piece = tid % a.nvec, tl = (tid / a.nvec) % a.tokens, hs = tid / group;
    const int tok = blockIdx.x * a.tokens + tl;
    const int D = a.cache.D, Hkv = a.cache.Hkv, QKVH = a.Hq + 2 * Hkv;
    const int h_end = min((int)(blockIdx.y + 1) * a.heads, QKVH);
    const int h0 = blockIdx.y * a.heads + hs;
    const bool active = hs < hpp && tok < a.token_num;

    // (T rows requested before the token's place is known: three dependent loads away)
    const T* in = static_cast<const T*>(a.qkv) + ((size_t)(active ? tok : 0) * QKVH) * D + piece * VEC;
    const T* bias = static_cast<const T*>(a.bias) + piece * VEC;
    Vec16<T> v[UNROLL], bv[UNROLL];
    auto request = [&](int hb) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int h = hb + u * hpp;
            if (active && h < h_end) {
                v[u] = load16_stream(in + (size_t)h * D);
                if (a.bias) bv[u] = load16(bias + (size_t)h * D);
            }
        }
    };
    request(h0);

    // Which sequence holds the thread's token: 64 sequences are looked at per step, a lane each, for all tokens of the workgroup -
    // their first tokens and histories come with the same round trip.
    const int lane = tid & (kWave - 1);
    int b = -1, first = 0, hist = 0;
    for (int c = 0; c < a.B; c += kWave) {
        const int s = min(c + lane, a.B - 1);
        const int start = a.cu[s], end = c + lane < a.B ? a.cu[s + 1] : 0x7FFFFFFF, before = a.hist[s];
        int mine = kWave;                            // sequences of this step that end at or before the token
        for (int i = 0; i < a.tokens; ++i) {
            const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(end <= (int)(blockIdx.x * a.tokens) + i));
            mine = i == tl ? n : mine;
        }
        const int from = min(mine, kWave - 1);
        const int f = __shfl(start, from, kWave), h = __shfl(before, from, kWave);
        if (b < 0 && mine < min(kWave, a.B - c)) {
            b = c + mine;
            first = f;
            hist = h;
        }
    }
    // behind the last sequence, or a sequence that is left alone
    if (!active || b < 0 || tok < first || hist < 0) return;
    const long long far = (long long)hist + ((long long)tok - first);
    // a position past what the table can hold has no page; its angle is still that of the position
    const int pos = far > 0x7FFFFFFF ? 0x7FFFFFFF : (int)far;
    const int page = page_of(a.cache, a.cache.table + (size_t)b * a.cache.max_pages, pos);
    const int npair = min(a.rotary_dim, D) / 2;
    float sn[VEC / 2], cs[VEC / 2];
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
        const int p = piece * (VEC / 2) + e;
        sn[e] = 0.f;
        cs[e] = 1.f;
        if (p < npair) rope_sincos(pos, rt.f[p], sn[e], cs[e]);
    }
    T* qo = static_cast<T*>(a.q_out) + (size_t)tok * a.q_stride + piece * VEC;
    const size_t row0 = page < 0 ? 0 : paged_offset(a.cache, page, 0, pos) + piece * VEC;
    const size_t head_step = (size_t)D << a.cache.page_shift;
    T* ko = static_cast<T*>(a.k_pages) + row0;
    T* vo = static_cast<T*>(a.v_pages) + row0;
    for (int hb = h0; hb < h_end; hb += hpp * UNROLL) {
        if (hb != h0) request(hb);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int h = hb + u * hpp;
            if (h >= h_end) break;
            float x[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = v[u].get(e);
            if (a.bias) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[e] += bv[u].get(e);
            }
            const bool rotate = h < a.Hq + Hkv;
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                // pairs past rotary_dim stay untouched bit for bit
                const bool on = rotate && piece * (VEC / 2) + e / 2 < npair;
                const float r0 = __builtin_fmaf(x[e], cs[e / 2], -(x[e + 1] * sn[e / 2]));
                const float r1 = __builtin_fmaf(x[e + 1], cs[e / 2], x[e] * sn[e / 2]);
                x[e] = on ? r0 : x[e];
                x[e + 1] = on ? r1 : x[e + 1];
            }
            Vec16<T> o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) o.set(e, x[e]);
            if (h < a.Hq) store16_stream(qo + (size_t)h * D, o);
            else if (page >= 0) store16_stream(h < a.Hq + Hkv ? ko + (h - a.Hq) * head_step : vo + (h - a.Hq - Hkv) * head_step, o);
        }
    }
}

}  // namespace
}  // namespace onellm

extern "C" int onellm_paged_qkv_store(int dtype, void* q_out, long q_stride, void* k_pages, void* v_pages, const void* qkv,
                                      const void* qkv_bias, const int* cu_tokens, const int* history_length, const int* block_table,
                                      int B, int token_num, int Hq, int Hkv, int D, int page_size, int num_pages, int max_pages,
                                      int layer, int num_layers, int rotary_dim, float rope_base, onellm_stream_t stream)
{
    using namespace onellm;
    const int rc = check_paged(dtype, k_pages, v_pages, block_table, B, Hq, Hkv, D, page_size, num_pages, max_pages, layer, num_layers);
    if (rc) return rc;
    if (token_num < 0 || !cu_tokens || !history_length) return ONELLM_EINVAL;
    if (rotary_dim < 0 || rotary_dim % 2 != 0 || (rotary_dim > 0 && !(rope_base > 0.f && rope_base < INFINITY))) return ONELLM_EINVAL;
    if (token_num == 0) return 0;
    if (!q_out || !qkv) return ONELLM_EINVAL;
    const int vec = dtype == ONELLM_FP16 ? 8 : 4, QKVH = Hq + 2 * Hkv;
    const size_t elt = 16 / vec;
    if (q_stride < (long)Hq * D) return ONELLM_EINVAL;
    if (token_num > 1 << 25) return ONELLM_EUNSUPPORTED;     // (four tokens or more per workgroup of 256: 2^31 threads, a launch takes below 2^32)
    if (!aligned16(q_out) || !aligned16(qkv) || (qkv_bias && !aligned16(qkv_bias)) || q_stride % vec != 0) return ONELLM_EUNSUPPORTED;
    // q_out may be qkv itself, q written over its own heads; any other overlap would be read after it was written
    const char *o0 = static_cast<const char*>(q_out), *i0 = static_cast<const char*>(qkv);
    const char *o1 = o0 + ((size_t)(token_num - 1) * q_stride + (size_t)Hq * D) * elt, *i1 = i0 + (size_t)token_num * QKVH * D * elt;
    const bool in_place = o0 == i0 && q_stride == (long)QKVH * D;
    if (!in_place && o0 < i1 && i0 < o1) return ONELLM_EINVAL;
    StoreArgs a;
    a.q_out = q_out;
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.qkv = qkv;
    a.bias = qkv_bias;
    a.cu = cu_tokens;
    a.hist = history_length;
    a.cache = make_paged(block_table, max_pages, num_pages, page_size, Hkv, D, layer);
    a.q_stride = q_stride;
    a.B = B;
    a.token_num = token_num;
    a.Hq = Hq;
    a.rotary_dim = rotary_dim;
    a.nvec = D / vec;
    a.tokens = 8;
    while (a.tokens * a.nvec > 256) a.tokens /= 2;
    // slices of the heads, until there are two workgroups per compute unit or a thread is down to one head (32 tokens, 48 heads
    // of 128: 10.6 us in one slice, 5.2 in 24)
    const int groups = (token_num + a.tokens - 1) / a.tokens, per_pass = 256 / (a.tokens * a.nvec);
    const int most = (QKVH + per_pass - 1) / per_pass, slices = groups >= 512 ? 1 : (512 / groups < most ? 512 / groups : most);
    a.heads = ((QKVH + slices - 1) / slices + per_pass - 1) / per_pass * per_pass;
    RopeTurns rt;
    fill_rope_turns(rt, D, rotary_dim, rope_base);
    const dim3 grid((token_num + a.tokens - 1) / a.tokens, (QKVH + a.heads - 1) / a.heads);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == ONELLM_FP16) hipLaunchKernelGGL((paged_qkv_store_kernel<__half>), grid, dim3(256), 0, st, a, rt);
    else hipLaunchKernelGGL((paged_qkv_store_kernel<float>), grid, dim3(256), 0, st, a, rt);
    return launch_status();
}
