// The paged key/value cache: new keys | values quantised into their pages, and read back as bf16.
//
// Pages are [page][kv head][row][d_kv], one f32 scale per (page, kv head, row) for the 8-bit types: a row of d_kv codes is contiguous and the
// rows of a page stand behind one another, so the attention reads whole pages of one head as one stream.  scale = max|x| / 127 (int8) or
// / 448 (e4m3) of the row, code = the nearest value of the type to x / scale in f32 (ties to even), kept within +-127 / +-448; a row of
// zeros has scale 0, a row with an infinity or a NaN has scale NaN and codes 0 (all of it reads back as NaN: nothing is hidden).
//
// Both kernels move bytes and nothing else: bound by memory.
#include "paged.h"
#include "rows.h"

namespace {

// A row of d_kv values is d_kv / 8 lanes; every lane takes two neighbouring tokens of its (head, key or value), whose loads are on their way
// before the first is used (80 x 58 tokens, 12 heads of 64, int8: written in 8.8 / 7.8 / 9.5 us and read back in 7.2 / 6.1 / 6.3 us with 1 / 2 / 4;
// 4 x 4000 tokens, 8 heads of 128 read back in 16.5 us = 5.4 TB/s).
constexpr int RPT = 2;

// x / s, correctly rounded, from the correctly rounded reciprocal of s (Markstein's final step: the remainder of the first quotient is exact in a
// fused multiply-add, so is its correction's rounding); a division proper costs three times the instructions and bound the kernel.
__device__ __forceinline__ float quotient(float x, float s, float inv) {
    const float q = x * inv;
    return fmaf(fmaf(-q, s, x), inv, q);
}

template <int T, int DK>
__global__ __launch_bounds__(256) void kv_write_kernel(const PagedSeqs s, const bf16_t* k, long long k_st, const bf16_t* v, long long v_st, unsigned char* kp,
                                                       unsigned char* vp, float* ks, float* vs, int H) {
    constexpr int LPR = DK / 8;
    const int b = blockIdx.y;
    const PagedSeq q = paged_seq(s, b);
    const long long row = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const int l = threadIdx.x % LPR;
    const int i0 = (int)(row / (2 * H)) * RPT, h2 = (int)(row % (2 * H));          // keys of all heads, then values of all heads
    const int n = min(q.nq, s.max_q) - i0;
    if (n <= 0) return;                                                            // (whole rows leave: the exchanges below stay within a row's lanes)
    const bool val = h2 >= H;
    const int h = val ? h2 - H : h2;
    const bf16_t* src = (val ? v + (size_t)(q.q0 + i0) * v_st : k + (size_t)(q.q0 + i0) * k_st) + h * DK + l * 8;
    const long long st = val ? v_st : k_st;
    uint4 raw[RPT];
    long long at[RPT];                                                             // cache row, or -1: nothing to write
#pragma unroll
    for (int j = 0; j < RPT; ++j) {
        const long long pos = (long long)q.len - q.nq + i0 + j;
        at[j] = -1;
        raw[j] = make_uint4(0, 0, 0, 0);
        if (j < n) {
            raw[j] = *reinterpret_cast<const uint4*>(src + j * st);
            const int pg = pos >= 0 && pos < q.len ? paged_page(s, b, (int)pos) : -1;
            if (pg >= 0) at[j] = (long long)((((size_t)pg * H + h) << s.page_shift) + (pos & ((1 << s.page_shift) - 1)));
        }
    }
#pragma unroll
    for (int j = 0; j < RPT; ++j) {
        unsigned char* dst = (val ? vp : kp) + ((size_t)at[j] * DK + l * 8) * KvType<T>::BYTES;
        if constexpr (T == VLT5_KV_BF16) {
            if (at[j] >= 0) *reinterpret_cast<uint4*>(dst) = raw[j];
        } else {
            constexpr float MOST = T == VLT5_KV_INT8 ? 127.f : 448.f;
            const uint32_t u[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
            float x[8], top = 0.f;
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = bf16_to_f32((bf16_t)(e & 1 ? u[e >> 1] >> 16 : u[e >> 1] & 0xffffu));
                bad |= !(fabsf(x[e]) <= 3.402823466e38f);
                top = fmaxf(top, fabsf(x[e]));
            }
            top = bad ? INFINITY : top;
#pragma unroll
            for (int o = 1; o < LPR; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
            const float sc = top == INFINITY ? __uint_as_float(0x7fc00000u) : top / MOST;
            const float inv = 1.0f / sc;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = quotient(x[e], sc, inv);
            if (!(sc >= 1e-30f)) {                                                 // a row of zeros, of NaN, or whose reciprocal would leave the range
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = sc > 0.f ? x[e] / sc : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_fmed3f(y[e], -MOST, MOST);
            uint2 out;
            if constexpr (T == VLT5_KV_INT8) {
                // 1.5 * 2^23 added: the sum's last place is 1, so the addition rounds to a whole number (ties to even) and its low byte is the code
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(y[e] + 12582912.0f);
#pragma unroll
                for (int e = 0; e < 8; e += 2) w[e] = __builtin_amdgcn_perm(w[e + 1], w[e], 0x0c0c0400u);
                out = make_uint2(w[0] | w[2] << 16, w[4] | w[6] << 16);
            } else {
                int w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
                w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w0, true);
                w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], w1, true);
                out = make_uint2((uint32_t)w0, (uint32_t)w1);
            }
            if (at[j] >= 0) {
                *reinterpret_cast<uint2*>(dst) = out;
                if (l == 0) (val ? vs : ks)[at[j]] = sc;
            }
        }
    }
}

// out [B][T][H * d_kv]: position t of every sequence, zeros at and past its length and where a page is not there.  Neighbouring positions
// 2 i, 2 i + 1 are in one page.
template <int T, int DK>
__global__ __launch_bounds__(256) void kv_read_kernel(const PagedSeqs s, const unsigned char* kp, const unsigned char* vp, const float* ks, const float* vs, int H,
                                                      int Tout, bf16_t* ko, bf16_t* vo) {
    constexpr int LPR = DK / 8;
    const int b = blockIdx.y;
    const long long row = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const int l = threadIdx.x % LPR;
    const int h2 = (int)(row % (2 * H));
    const long long t4 = row / (2 * H) * RPT;
    if (t4 >= Tout) return;
    const int t = (int)t4;
    const bool val = h2 >= H;
    const int h = val ? h2 - H : h2;
    const int len = paged_seq(s, b).len;
    const int pg = t < len ? paged_page(s, b, t) : -1;
    const size_t at = (((size_t)max(pg, 0) * H + h) << s.page_shift) + (t & ((1 << s.page_shift) - 1));
    bf16_t* dst = (val ? vo : ko) + (((size_t)b * Tout + t) * H + h) * DK + l * 8;
    uint4 out[RPT] = {};
    if (pg >= 0) {
        const unsigned char* src = (val ? vp : kp) + (at * DK + l * 8) * KvType<T>::BYTES;
        if constexpr (T == VLT5_KV_BF16) {
#pragma unroll
            for (int j = 0; j < RPT; ++j) out[j] = *reinterpret_cast<const uint4*>(src + j * DK * 2);
        } else {
            uint2 c[RPT];
#pragma unroll
            for (int j = 0; j < RPT; ++j) c[j] = *reinterpret_cast<const uint2*>(src + j * DK);
            const float2 s2 = *reinterpret_cast<const float2*>((val ? vs : ks) + at);
            const float sc[RPT] = {s2.x, s2.y};
#pragma unroll
            for (int j = 0; j < RPT; ++j) {
                const uint2 p0 = codes_to_bf16<T>(c[j].x), p1 = codes_to_bf16<T>(c[j].y);
                const uint32_t p[4] = {p0.x, p0.y, p1.x, p1.y};
                uint32_t r[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = pack_bf16x2(__uint_as_float(p[e] << 16) * sc[j], __uint_as_float(p[e] & 0xffff0000u) * sc[j]);   // to f32, then to bf16
                out[j] = make_uint4(r[0], r[1], r[2], r[3]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < RPT; ++j)
        if (t + j < Tout) *reinterpret_cast<uint4*>(dst + (size_t)j * H * DK) = t + j < len ? out[j] : make_uint4(0, 0, 0, 0);
}

}  // namespace

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
    const long long rows = ((long long)s.max_q + RPT - 1) / RPT * 2 * c->n_kv_heads;
    const long long blocks = (rows * (c->d_kv / 8) + 255) / 256;
    if (blocks * 256 > VLT5_MOST_THREADS) return VLT5_ERR_ARG;
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
    const long long blocks = (((long long)T + RPT - 1) / RPT * 2 * c->n_kv_heads * (c->d_kv / 8) + 255) / 256;
    if (blocks * 256 > VLT5_MOST_THREADS) return VLT5_ERR_ARG;
    const dim3 grid((unsigned)blocks, s.B);
#define KVR(TY, D) hipLaunchKernelGGL((kv_read_kernel<TY, D>), grid, dim3(256), 0, (hipStream_t)stream, s, (const unsigned char*)c->k, (const unsigned char*)c->v, \
                                      c->k_scale, c->v_scale, c->n_kv_heads, T, (bf16_t*)k_out, (bf16_t*)v_out)
    KV_DISPATCH(KVR);
#undef KVR
    LAUNCH_CHECK();
    return VLT5_OK;
}
