// The paged key/value cache: new keys | values quantised into their pages, and read back as bf16.
//
// Pages are [page][kv head][row][d_kv], one f32 scale per (page, kv head, row) for the 8-bit types: a row of d_kv codes is contiguous and the
// rows of a page stand behind one another, so the attention reads whole pages of one head as one stream.  scale = max|x| / 127 (int8) or
// / 448 (e4m3) of the row, code = the nearest value of the type to x / scale in f32 (ties to even), kept within +-127 / +-448; a row of
// zeros has scale 0, a row with an infinity or a NaN has scale NaN and codes 0 (all of it reads back as NaN: nothing is hidden).
//
// Both kernels move bytes and nothing else: bound by memory.
#include "paged.h"

namespace {

template <int T, int DK>
__global__ __launch_bounds__(256) void kv_write_kernel(const PagedSeqs s, const bf16_t* k, long long k_st, const bf16_t* v, long long v_st, unsigned char* kp,
                                                       unsigned char* vp, float* ks, float* vs, int H) {
    constexpr int LPR = DK / 8;                                               // lanes of a row, eight values each
    const int b = blockIdx.y;
    const PagedSeq q = paged_seq(s, b);
    const int row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, l = threadIdx.x % LPR;
    const int i = row / (2 * H), h2 = row % (2 * H);                          // keys of all heads, then values of all heads
    if (i >= min(q.nq, s.max_q)) return;                                      // (whole rows leave: the exchanges below stay within a row's lanes)
    const long long pos = (long long)q.len - q.nq + i;
    if (pos < 0 || pos >= q.len) return;
    const int pg = paged_page(s, b, (int)pos);
    if (pg < 0) return;
    const bool val = h2 >= H;
    const int h = val ? h2 - H : h2;
    const bf16_t* src = (val ? v + (size_t)(q.q0 + i) * v_st : k + (size_t)(q.q0 + i) * k_st) + h * DK + l * 8;
    const size_t at = (((size_t)pg * H + h) << s.page_shift) + (pos & ((1 << s.page_shift) - 1));
    const uint4 raw = *reinterpret_cast<const uint4*>(src);
    unsigned char* dst = (val ? vp : kp) + (at * DK + l * 8) * KvType<T>::BYTES;
    if constexpr (T == VLT5_KV_BF16) {
        *reinterpret_cast<uint4*>(dst) = raw;
    } else {
        constexpr float MOST = T == VLT5_KV_INT8 ? 127.f : 448.f;
        const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
        float x[8], top = 0.f;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = bf16_to_f32((bf16_t)(e & 1 ? u[e >> 1] >> 16 : u[e >> 1] & 0xffffu));
            bad |= !(fabsf(x[e]) <= 3.402823466e38f);
            top = fmaxf(top, fabsf(x[e]));
        }
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) {
            top = fmaxf(top, __shfl_xor(top, o, 64));
            bad |= __shfl_xor((int)bad, o, 64) != 0;
        }
        const float sc = bad ? __uint_as_float(0x7fc00000u) : top / MOST;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = sc > 0.f ? fminf(fmaxf(x[e] / sc, -MOST), MOST) : 0.f;
        uint2 out;
        if constexpr (T == VLT5_KV_INT8) {
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e >> 2] |= ((uint32_t)(int)rintf(y[e]) & 0xffu) << (8 * (e & 3));
            out = make_uint2(w[0], w[1]);
        } else {
            int w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
            w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w0, true);
            w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], w1, true);
            out = make_uint2((uint32_t)w0, (uint32_t)w1);
        }
        *reinterpret_cast<uint2*>(dst) = out;
        if (l == 0) (val ? vs : ks)[at] = sc;
    }
}

// out [B][T][H * d_kv]: position t of every sequence, zeros at and past its length and where a page is not there
template <int T, int DK>
__global__ __launch_bounds__(256) void kv_read_kernel(const PagedSeqs s, const unsigned char* kp, const unsigned char* vp, const float* ks, const float* vs, int H,
                                                      int Tout, bf16_t* ko, bf16_t* vo) {
    constexpr int LPR = DK / 8;
    const int b = blockIdx.y;
    const long long row = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const int l = threadIdx.x % LPR;
    const int h = (int)(row % H);
    const long long tv = row / H;                                              // keys of all positions, then values of all positions
    if (tv >= 2LL * Tout) return;
    const bool val = tv >= Tout;
    const int t = (int)(val ? tv - Tout : tv);
    const PagedSeq q = paged_seq(s, b);
    uint4 out = make_uint4(0, 0, 0, 0);
    const int pg = t < q.len ? paged_page(s, b, t) : -1;
    if (pg >= 0) {
        const size_t at = (((size_t)pg * H + h) << s.page_shift) + (t & ((1 << s.page_shift) - 1));
        const unsigned char* src = (val ? vp : kp) + (at * DK + l * 8) * KvType<T>::BYTES;
        if constexpr (T == VLT5_KV_BF16) {
            out = *reinterpret_cast<const uint4*>(src);
        } else {
            const uint2 c = *reinterpret_cast<const uint2*>(src);
            const float sc = (val ? vs : ks)[at];
            const uint2 p0 = codes_to_bf16<T>(c.x), p1 = codes_to_bf16<T>(c.y);
            const uint32_t p[4] = {p0.x, p0.y, p1.x, p1.y};
            uint32_t r[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = pack_bf16x2(__uint_as_float(p[e] << 16) * sc, __uint_as_float(p[e] & 0xffff0000u) * sc);   // exact codes: one rounding
            out = make_uint4(r[0], r[1], r[2], r[3]);
        }
    }
    *reinterpret_cast<uint4*>((val ? vo : ko) + (((size_t)b * Tout + t) * H + h) * DK + l * 8) = out;
}

}  // namespace

// host-side checks shared by the entry points of the cache
int vlt5_paged_check(const vlt5_paged_kv* c, const vlt5_paged_seqs* q) {
    if (!c || !q || !c->k || !c->v || !q->table || !q->kv_lens) return VLT5_ERR_ARG;
    if (c->type != VLT5_KV_BF16 && c->type != VLT5_KV_INT8 && c->type != VLT5_KV_FP8) return VLT5_ERR_ARG;
    if (c->type != VLT5_KV_BF16 && (!c->k_scale || !c->v_scale)) return VLT5_ERR_ARG;
    if (c->n_pages <= 0 || c->n_kv_heads <= 0 || c->n_kv_heads > 1024 || (c->d_kv != 64 && c->d_kv != 128)) return VLT5_ERR_ARG;
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) return VLT5_ERR_ARG;
    if (q->B <= 0 || q->B > 65535 || q->max_pages <= 0 || q->n_tok < 0 || q->max_q < 0) return VLT5_ERR_ARG;
    if (!q->cu_q && q->n_tok != 0 && q->n_tok != q->B) return VLT5_ERR_ARG;
    if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 15) return VLT5_ERR_ALIGN;
    return VLT5_OK;
}
PagedSeqs vlt5_paged_seqs_of(const vlt5_paged_kv* c, const vlt5_paged_seqs* q) {
    PagedSeqs s;
    s.table = q->table; s.max_pages = q->max_pages; s.page_shift = __builtin_ctz(c->page_size); s.n_pages = c->n_pages;
    s.lens = q->kv_lens; s.cu = q->cu_q; s.B = q->B; s.n_tok = q->n_tok;
    s.max_q = q->cu_q ? (q->max_q > 0 && q->max_q < q->n_tok ? q->max_q : q->n_tok) : 1;
    return s;
}

#define KV_DISPATCH(F)                                                                                                                  \
    do {                                                                                                                                \
        if (c->d_kv == 64) {                                                                                                            \
            if (c->type == VLT5_KV_BF16) F(VLT5_KV_BF16, 64); else if (c->type == VLT5_KV_INT8) F(VLT5_KV_INT8, 64); else F(VLT5_KV_FP8, 64);     \
        } else {                                                                                                                        \
            if (c->type == VLT5_KV_BF16) F(VLT5_KV_BF16, 128); else if (c->type == VLT5_KV_INT8) F(VLT5_KV_INT8, 128); else F(VLT5_KV_FP8, 128);  \
        }                                                                                                                               \
    } while (0)

extern "C" int vlt5_kv_page_write(const vlt5_paged_kv* c, const vlt5_paged_seqs* q, const void* k, long long k_st, const void* v, long long v_st, void* stream) {
    const int rc = vlt5_paged_check(c, q);
    if (rc) return rc;
    if (!k || !v || k_st < (long long)c->n_kv_heads * c->d_kv || v_st < (long long)c->n_kv_heads * c->d_kv) return VLT5_ERR_ARG;
    if ((k_st & 7) || (v_st & 7) || (((uintptr_t)k | (uintptr_t)v) & 15)) return VLT5_ERR_ALIGN;
    if (q->n_tok == 0) return VLT5_OK;
    const PagedSeqs s = vlt5_paged_seqs_of(c, q);
    const long long rows = (long long)s.max_q * 2 * c->n_kv_heads;
    const long long blocks = (rows * (c->d_kv / 8) + 255) / 256;
    if (rows > 0x7fffffffLL || blocks > 0x7fffffffLL) return VLT5_ERR_ARG;
    const dim3 grid((unsigned)blocks, s.B);
#define KVW(T, D) hipLaunchKernelGGL((kv_write_kernel<T, D>), grid, dim3(256), 0, (hipStream_t)stream, s, (const bf16_t*)k, k_st, (const bf16_t*)v, v_st, \
                                     (unsigned char*)c->k, (unsigned char*)c->v, c->k_scale, c->v_scale, c->n_kv_heads)
    KV_DISPATCH(KVW);
#undef KVW
    LAUNCH_CHECK();
    return VLT5_OK;
}

extern "C" int vlt5_kv_page_read(const vlt5_paged_kv* c, const vlt5_paged_seqs* q, int T, void* k_out, void* v_out, void* stream) {
    const int rc = vlt5_paged_check(c, q);
    if (rc) return rc;
    if (!k_out || !v_out || T < 0) return VLT5_ERR_ARG;
    if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) return VLT5_ERR_ALIGN;
    if (T == 0) return VLT5_OK;
    const PagedSeqs s = vlt5_paged_seqs_of(c, q);
    const long long blocks = (2LL * T * c->n_kv_heads * (c->d_kv / 8) + 255) / 256;
    if (blocks > 0x7fffffffLL) return VLT5_ERR_ARG;
    const dim3 grid((unsigned)blocks, s.B);
#define KVR(TY, D) hipLaunchKernelGGL((kv_read_kernel<TY, D>), grid, dim3(256), 0, (hipStream_t)stream, s, (const unsigned char*)c->k, (const unsigned char*)c->v, \
                                      c->k_scale, c->v_scale, c->n_kv_heads, T, (bf16_t*)k_out, (bf16_t*)v_out)
    KV_DISPATCH(KVR);
#undef KVR
    LAUNCH_CHECK();
    return VLT5_OK;
}
