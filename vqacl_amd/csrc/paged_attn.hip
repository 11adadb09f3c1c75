// Attention of the newest tokens of every sequence over its paged cache: softmax(scale * q K^T + bias) V, single tokens and chunks.
//
// The query rows of one (sequence, kv head) are the tokens times the query heads that share the kv head, sixteen of them a tile.  Keys are
// walked in tiles of 64 with the running maximum and sum of the softmax in f32, and everything stays in registers:
//   scores  S^T[key, row] = mfma(A = 16 keys, B = 16 query rows): a lane ends up with four consecutive keys of ONE row (row = lane % 16);
//   output  O^T[d, row] += mfma(A = V^T, B = P^T): the 32 keys of one instruction may be taken in any order as long as both operands agree,
//           so the eight keys of a lane's B operand are simply the ones it has scores of -- no exchange between lanes -- and the A operand is
//           built from the same eight rows of V, d_kv / 16 neighbouring values of each: the conversion to bf16 pairs them by key, which IS
//           the transposition.
// 8-bit codes are exact in bf16; the scale of a key multiplies its score, the scale of a value its probability (in f32, before the one
// rounding of the probabilities to bf16).
#include "paged.h"

namespace {

struct PagedAttnArgs {
    PagedSeqs s;
    const unsigned char* k; const unsigned char* v; const float* ks; const float* vs;
    const bf16_t* q; long long q_st;
    bf16_t* out; long long o_st;
    float* lse;                               // [n_tok][H] or null
    int H, Hkv, g;
    float scale;
    int causal;
    const float* bias; int nd;                // [H][nd] by distance, the last entry for everything further
    int row_tiles, splits;
    float* part_o; float* part_ml;            // [splits][n_tok * H][d_kv], [splits][n_tok * H][2]
};

constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// one lane's four consecutive dwords / pairs of a row of codes as MFMA operands
template <int T, int DK>
__device__ __forceinline__ void load_key_frags(const unsigned char* row, int kq, bf16x8_t (&f)[DK / 32]) {
    if constexpr (T == VLT5_KV_BF16) {
#pragma unroll
        for (int i = 0; i < DK / 32; ++i) f[i] = *reinterpret_cast<const bf16x8_t*>(row + (i * 32 + kq * 8) * 2);
    } else {
#pragma unroll
        for (int c = 0; c < DK / 64; ++c) {
            const uint4 u = *reinterpret_cast<const uint4*>(row + c * 64 + kq * 16);
            const uint2 a = codes_to_bf16<T>(u.x), b = codes_to_bf16<T>(u.y), e = codes_to_bf16<T>(u.z), d = codes_to_bf16<T>(u.w);
            f[c * 2] = __builtin_bit_cast(bf16x8_t, make_uint4(a.x, a.y, b.x, b.y));
            f[c * 2 + 1] = __builtin_bit_cast(bf16x8_t, make_uint4(e.x, e.y, d.x, d.y));
        }
    }
}
// ... and the query row in the same order of d
template <int T, int DK>
__device__ __forceinline__ void load_query_frags(const bf16_t* row, int kq, bf16x8_t (&f)[DK / 32]) {
#pragma unroll
    for (int i = 0; i < DK / 32; ++i) {
        const int d = T == VLT5_KV_BF16 ? i * 32 + kq * 8 : (i >> 1) * 64 + kq * 16 + (i & 1) * 8;
        f[i] = *reinterpret_cast<const bf16x8_t*>(row + d);
    }
}
// DK / 16 neighbouring values of a row of V, raw
template <int T, int DK> struct VRow { uint32_t w[DK / 16 * KvType<T>::BYTES / 4]; };
template <int T, int DK>
__device__ __forceinline__ VRow<T, DK> load_vrow(const unsigned char* p) {
    VRow<T, DK> r;
    constexpr int N = DK / 16 * KvType<T>::BYTES / 4;
    if constexpr (N == 1) r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (N == 2) { const uint2 u = *reinterpret_cast<const uint2*>(p); r.w[0] = u.x; r.w[1] = u.y; }
    else { const uint4 u = *reinterpret_cast<const uint4*>(p); r.w[0] = u.x; r.w[1] = u.y; r.w[2] = u.z; r.w[3] = u.w; }
    return r;
}
// value j of rows a and b as a bf16 pair
template <int T, int DK>
__device__ __forceinline__ uint32_t vpair(const VRow<T, DK>& a, const VRow<T, DK>& b, int j) {
    if constexpr (T == VLT5_KV_BF16) {
        return __builtin_amdgcn_perm(b.w[j >> 1], a.w[j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
    } else if constexpr (T == VLT5_KV_INT8) {
        return pack_bf16x2(sbyte(a.w[j >> 2], j & 3), sbyte(b.w[j >> 2], j & 3));
    } else {
        const uint32_t m = __builtin_amdgcn_perm(b.w[j >> 2], a.w[j >> 2], j & 2 ? 0x07030602u : 0x05010400u);
        return cvt_fp8_pair(m, j & 1);
    }
}

template <int T, int DK, int NW>
__global__ __launch_bounds__(NW * 64) void paged_attn_kernel(const PagedAttnArgs a) {
    constexpr int NF = DK / 32, ND = DK / 16, ROWB = DK * KvType<T>::BYTES;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4;
    int id = blockIdx.x;
    const int sp = id % a.splits; id /= a.splits;
    const int rt = id % a.row_tiles; id /= a.row_tiles;
    const int hk = id % a.Hkv, b = id / a.Hkv;
    const PagedSeq sq = paged_seq(a.s, b);
    const int rows = min(sq.nq, a.s.max_q) * a.g;
    if (rt * 16 >= rows) return;
    const int r = min(rt * 16 + r16, rows - 1);
    const int tok = r / a.g, hq = hk * a.g + r % a.g;
    const int pos = sq.len - sq.nq + tok;                                          // this row's position (negative: more new tokens than keys)
    const int L = a.causal ? min(pos + 1, sq.len) : sq.len;                       // keys this row sees
    const int first = sq.len - sq.nq + rt * 16 / a.g, last = sq.len - sq.nq + min(rt * 16 + 15, rows - 1) / a.g;
    const int Lmin = a.causal ? first + 1 : sq.len, Lmax = max(a.causal ? last + 1 : sq.len, 0);
    const int per = ((Lmax + a.splits - 1) / a.splits + 63) & ~63;
    const int lo = min(sp * per, Lmax), hi = min(lo + per, Lmax);

    bf16x8_t fq[NF];
    load_query_frags<T, DK>(a.q + (size_t)(sq.q0 + tok) * a.q_st + hq * DK, kq, fq);
    const float* bias = a.bias ? a.bias + (size_t)hq * a.nd : nullptr;

    f32x4_t o[ND];
#pragma unroll
    for (int j = 0; j < ND; ++j) o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    for (int t0 = lo + w * 64; t0 < hi; t0 += NW * 64) {
        size_t base[4];
        bool there[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pg = t0 + i * 16 < hi ? paged_page(a.s, b, t0 + i * 16) : -1;
            there[i] = pg >= 0;
            base[i] = (((size_t)max(pg, 0) * a.Hkv + hk) << a.s.page_shift) + ((t0 + i * 16) & ((1 << a.s.page_shift) - 1));
        }
        const bool whole = t0 + 64 <= min(Lmin, hi) && there[0] && there[1] && there[2] && there[3];
        VRow<T, DK> vr[4][4];
        float4 kscale[4], vscale[4];
        f32x4_t sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bf16x8_t fk[NF];
            load_key_frags<T, DK>(a.k + (base[i] + r16) * ROWB, kq, fk);
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[i][e] = load_vrow<T, DK>(a.v + (base[i] + kq * 4 + e) * ROWB + r16 * (ROWB / 16));
            kscale[i] = vscale[i] = make_float4(1.f, 1.f, 1.f, 1.f);
            if constexpr (KvType<T>::SCALED) {
                kscale[i] = *reinterpret_cast<const float4*>(a.ks + base[i] + kq * 4);
                vscale[i] = *reinterpret_cast<const float4*>(a.vs + base[i] + kq * 4);
            }
            sc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < NF; ++f) sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fk[f], fq[f], sc[i], 0, 0, 0);
        }
        float p[4][4], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float kk[4] = {kscale[i].x, kscale[i].y, kscale[i].z, kscale[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = t0 + i * 16 + kq * 4 + e;
                float s = sc[i][e] * (kk[e] * a.scale);
                if (bias) s += bias[min(max(pos - t, 0), a.nd - 1)];
                if (!whole) s = there[i] && t < L ? s : -INFINITY;
                p[i][e] = s;
                top = fmaxf(top, s);
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float mn = fmaxf(m, top), ms = mn == -INFINITY ? 0.f : mn;            // a row that has seen no key yet stays at -inf, sum 0
        const float fix = exp2_hw((m - ms) * LOG2E);
        m = mn;
        l *= fix;
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] *= fix;
        uint32_t pb[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float vv[4] = {vscale[i].x, vscale[i].y, vscale[i].z, vscale[i].w};
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float pe = exp2_hw((p[i][e] - ms) * LOG2E);
                l += pe;
                x[e] = pe * vv[e];
                if (!whole) {                                                        // what lies behind the last key may hold anything, NaN too
                    const bool in = there[i] && t0 + i * 16 + kq * 4 + e < sq.len;
                    if (!(in && t0 + i * 16 + kq * 4 + e < L)) x[e] = 0.f;
                    if (!in) vr[i][e] = VRow<T, DK>{};
                }
            }
            pb[i][0] = pack_bf16x2(x[0], x[1]);
            pb[i][1] = pack_bf16x2(x[2], x[3]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bf16x8_t fp = __builtin_bit_cast(bf16x8_t, make_uint4(pb[2 * h][0], pb[2 * h][1], pb[2 * h + 1][0], pb[2 * h + 1][1]));
#pragma unroll
            for (int j = 0; j < ND; ++j) {
                const uint4 fv = make_uint4(vpair<T, DK>(vr[2 * h][0], vr[2 * h][1], j), vpair<T, DK>(vr[2 * h][2], vr[2 * h][3], j),
                                            vpair<T, DK>(vr[2 * h + 1][0], vr[2 * h + 1][1], j), vpair<T, DK>(vr[2 * h + 1][2], vr[2 * h + 1][3], j));
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, fv), fp, o[j], 0, 0, 0);
            }
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // ---- the waves' shares of the keys meet in LDS, always in the order of the waves ----
    __shared__ float so[NW][16][DK + 4];
    __shared__ float sm[NW][16], sl[NW][16];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < ND; ++j) so[w][r16][(kq * 4 + e) * ND + j] = o[j][e];      // row of the A operand (kq * 4 + e) stands for d = that * ND + j
    if (lane < 16) { sm[w][lane] = m; sl[w][lane] = l; }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (DK / 4); i += NW * 64) {
        const int rr = i / (DK / 4), d = i % (DK / 4) * 4;
        if (rt * 16 + rr >= rows) continue;
        float mx = sm[0][rr];
#pragma unroll
        for (int ww = 1; ww < NW; ++ww) mx = fmaxf(mx, sm[ww][rr]);
        const float ms = mx == -INFINITY ? 0.f : mx;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int ww = 0; ww < NW; ++ww) {
            const float f = exp2_hw((sm[ww][rr] - ms) * LOG2E);
            const float4 x = *reinterpret_cast<const float4*>(&so[ww][rr][d]);
            sum += sl[ww][rr] * f;
            acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
        }
        const int tk = (rt * 16 + rr) / a.g, hh = hk * a.g + (rt * 16 + rr) % a.g;
        const size_t token = (size_t)(sq.q0 + tk);
        if (a.splits == 1) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            *reinterpret_cast<uint2*>(a.out + token * a.o_st + hh * DK + d) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
            if (a.lse && d == 0) a.lse[token * a.H + hh] = sum == 0.f ? -INFINITY : mx + logf(sum);
        } else {
            const size_t at = ((size_t)sp * a.s.n_tok + token) * a.H + hh;
            *reinterpret_cast<float4*>(a.part_o + at * DK + d) = acc;
            if (d == 0) { a.part_ml[at * 2] = mx; a.part_ml[at * 2 + 1] = sum; }
        }
    }
}

// joins the splits of a row, in their order
template <int DK>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttnArgs a) {
    int id = blockIdx.x;
    const int rt = id % a.row_tiles; id /= a.row_tiles;
    const int hk = id % a.Hkv, b = id / a.Hkv;
    const PagedSeq sq = paged_seq(a.s, b);
    const int rows = min(sq.nq, a.s.max_q) * a.g;
    for (int i = threadIdx.x; i < 16 * (DK / 4); i += 256) {
        const int rr = rt * 16 + i / (DK / 4), d = i % (DK / 4) * 4;
        if (rr >= rows) continue;
        const size_t row = (size_t)(sq.q0 + rr / a.g) * a.H + hk * a.g + rr % a.g;
        const size_t step = (size_t)a.s.n_tok * a.H;
        float mx = -INFINITY;
        for (int sp = 0; sp < a.splits; ++sp) mx = fmaxf(mx, a.part_ml[(sp * step + row) * 2]);
        const float ms = mx == -INFINITY ? 0.f : mx;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
        for (int sp = 0; sp < a.splits; ++sp) {
            const float f = exp2_hw((a.part_ml[(sp * step + row) * 2] - ms) * LOG2E);
            const float4 x = *reinterpret_cast<const float4*>(a.part_o + (sp * step + row) * DK + d);
            sum += a.part_ml[(sp * step + row) * 2 + 1] * f;
            acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint2*>(a.out + (row / a.H) * a.o_st + (row % a.H) * DK + d) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
        if (a.lse && d == 0) a.lse[row] = sum == 0.f ? -INFINITY : mx + logf(sum);
    }
}

// how many workgroups share the keys of a row tile: enough to fill the chip, no share below 512 keys
int paged_splits(const vlt5_paged_attn_desc* d, int row_tiles) {
    const long long most_kv = d->max_kv > 0 ? d->max_kv : (long long)d->seqs.max_pages * d->kv.page_size;
    const long long tiles = (long long)d->seqs.B * d->kv.n_kv_heads * row_tiles;
    long long sp = (1024 + tiles - 1) / tiles;
    sp = sp < most_kv / 512 ? sp : most_kv / 512;
    return (int)(sp < 1 ? 1 : (sp > 64 ? 64 : sp));
}
int paged_row_tiles(const PagedSeqs& s, int g) { return (int)(((long long)s.max_q * g + 15) / 16); }

}  // namespace

int vlt5_paged_check(const vlt5_paged_kv* c, const vlt5_paged_seqs* q);
PagedSeqs vlt5_paged_seqs_of(const vlt5_paged_kv* c, const vlt5_paged_seqs* q);

extern "C" long long vlt5_paged_attn_workspace_bytes(const vlt5_paged_attn_desc* d) {
    if (!d || vlt5_paged_check(&d->kv, &d->seqs) || d->H <= 0 || d->H % d->kv.n_kv_heads) return -1;
    const PagedSeqs s = vlt5_paged_seqs_of(&d->kv, &d->seqs);
    const int sp = paged_splits(d, paged_row_tiles(s, d->H / d->kv.n_kv_heads));
    return sp == 1 ? 0 : (long long)sp * s.n_tok * d->H * (d->kv.d_kv + 2) * 4;
}

extern "C" int vlt5_paged_attn(const vlt5_paged_attn_desc* d, void* stream) {
    if (!d || !d->q || !d->out) return VLT5_ERR_ARG;
    const int rc = vlt5_paged_check(&d->kv, &d->seqs);
    if (rc) return rc;
    const vlt5_paged_kv& c = d->kv;
    if (d->H <= 0 || d->H % c.n_kv_heads || d->H > 1024) return VLT5_ERR_ARG;
    if (d->q_st < (long long)d->H * c.d_kv || d->o_st < (long long)d->H * c.d_kv) return VLT5_ERR_ARG;
    if (d->rel_bias && (d->n_dist <= 0 || !d->causal)) return VLT5_ERR_ARG;
    if ((d->q_st & 7) || (d->o_st & 7) || (((uintptr_t)d->q | (uintptr_t)d->out | (uintptr_t)d->workspace) & 15)) return VLT5_ERR_ALIGN;
    if (d->seqs.n_tok == 0) return VLT5_OK;
    PagedAttnArgs a;
    a.s = vlt5_paged_seqs_of(&c, &d->seqs);
    a.k = (const unsigned char*)c.k; a.v = (const unsigned char*)c.v; a.ks = c.k_scale; a.vs = c.v_scale;
    a.q = (const bf16_t*)d->q; a.q_st = d->q_st; a.out = (bf16_t*)d->out; a.o_st = d->o_st; a.lse = d->lse;
    a.H = d->H; a.Hkv = c.n_kv_heads; a.g = d->H / c.n_kv_heads;
    a.scale = d->scale; a.causal = d->causal; a.bias = d->rel_bias; a.nd = d->n_dist;
    a.row_tiles = paged_row_tiles(a.s, a.g);
    a.splits = paged_splits(d, a.row_tiles);
    const long long rows = (long long)a.s.n_tok * a.H;
    if (a.splits > 1) {
        if (!d->workspace || d->workspace_bytes < (long long)a.splits * rows * (c.d_kv + 2) * 4) return VLT5_ERR_ARG;
        a.part_o = (float*)d->workspace;
        a.part_ml = a.part_o + (size_t)a.splits * rows * c.d_kv;
    } else {
        a.part_o = a.part_ml = nullptr;
    }
    const long long tiles = (long long)a.s.B * a.Hkv * a.row_tiles;
    if (tiles * a.splits > 0x7fffffffLL) return VLT5_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
#define PA(T, D) hipLaunchKernelGGL((paged_attn_kernel<T, D, 4>), dim3((unsigned)(tiles * a.splits)), dim3(256), 0, st, a)
    if (c.d_kv == 64) {
        if (c.type == VLT5_KV_BF16) PA(VLT5_KV_BF16, 64); else if (c.type == VLT5_KV_INT8) PA(VLT5_KV_INT8, 64); else PA(VLT5_KV_FP8, 64);
    } else {
        if (c.type == VLT5_KV_BF16) PA(VLT5_KV_BF16, 128); else if (c.type == VLT5_KV_INT8) PA(VLT5_KV_INT8, 128); else PA(VLT5_KV_FP8, 128);
    }
#undef PA
    LAUNCH_CHECK();
    if (a.splits > 1) {
        if (c.d_kv == 64) hipLaunchKernelGGL(paged_join_kernel<64>, dim3((unsigned)tiles), dim3(256), 0, st, a);
        else hipLaunchKernelGGL(paged_join_kernel<128>, dim3((unsigned)tiles), dim3(256), 0, st, a);
        LAUNCH_CHECK();
    }
    return VLT5_OK;
}
