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
    int row_tiles, join_tiles, splits;
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

// ---- chunks: many rows share the keys ------------------------------------------------------------------------------------------------
// 128 query rows a workgroup, 32 of them a wave; tiles of 64 keys and values are converted to bf16 ONCE per workgroup on their way into LDS
// (two buffers: the next tile's loads are in flight while one is used), the same two products as above on 32 x 32 x 16 instructions.
//   K in LDS: rows of d_kv values + 16 bytes, so that 16 rows of an operand start in 16 bank groups;
//   V in LDS: in the order the operand wants it, [16 keys][d % NT][lane] pieces of eight keys of one d -- the thread that loaded d_kv / 32
//   neighbouring values of eight rows pairs them by key; d = NT * m + j for row m of operand tile j makes its stores and the reads consecutive.
// The running maximum moves only when a row's new one is more than 2^8 away: until then probabilities up to 256 are exact enough in every
// type they pass through (f32 sums, bf16 relative to the value), and the output's 16 * NT registers are left alone.
typedef __attribute__((ext_vector_type(16))) float f32x16_t;

template <int T, int DK, bool BIAS>
__global__ __launch_bounds__(256, 2) void paged_chunk_kernel(const PagedAttnArgs a) {
    constexpr int NT = DK / 32, NKS = DK / 16, BY = KvType<T>::BYTES, ROWB = DK * BY;
    constexpr int KROW = DK * 2 + 16, KBYTES = 64 * KROW, VBYTES = 4 * NT * 1024, BUF = KBYTES + VBYTES + 512;
    constexpr int KCH = ROWB / 16, KP = 64 * KCH / 256;                                 // 16-byte pieces of a key row; pieces of a thread
    constexpr int VW = (NT * BY + 3) / 4;                                               // dwords of a thread's share of a value row
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r32 = lane & 31, h = lane >> 5;
    const int pairs = a.s.B * a.Hkv;
    const int pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
    const int sp = rest % a.splits, rt = a.row_tiles - 1 - rest / a.splits;             // the last rows see the most keys: they start first
    const int hk = pair % a.Hkv, b = pair / a.Hkv;
    const PagedSeq sq = paged_seq(a.s, b);
    const int rows = min(sq.nq, a.s.max_q) * a.g;
    if (rt * 128 >= rows) return;
    const int wr0 = rt * 128 + w * 32;                                                  // first row of the wave
    const int r = min(wr0 + r32, rows - 1);
    const int tok = r / a.g, hq = hk * a.g + r % a.g;
    const int pos = sq.len - sq.nq + tok;
    const int L = a.causal ? min(pos + 1, sq.len) : sq.len;
    const int p0 = sq.len - sq.nq;
    const int Lmax = max(a.causal ? p0 + min(rt * 128 + 127, rows - 1) / a.g + 1 : sq.len, 0);
    const int wLmin = a.causal ? p0 + min(wr0, rows - 1) / a.g + 1 : sq.len;            // the wave's rows all see the keys below this ...
    const int wLmax = wr0 < rows ? (a.causal ? p0 + min(wr0 + 31, rows - 1) / a.g + 1 : sq.len) : 0;      // ... and none those from here on
    const int per = ((Lmax + a.splits - 1) / a.splits + 63) & ~63;
    const int lo = min(sp * per, Lmax), hi = min(lo + per, Lmax);

    bf16x8_t fq[NKS];
    const bf16_t* qrow = a.q + (size_t)(sq.q0 + tok) * a.q_st + hq * DK;
#pragma unroll
    for (int i = 0; i < NKS; ++i) fq[i] = *reinterpret_cast<const bf16x8_t*>(qrow + i * 16 + h * 8);
    const float* bias = BIAS ? a.bias + (size_t)hq * a.nd : nullptr;
    const float unit = BIAS ? 1.f : LOG2E;                                              // without a bias scores are kept in powers of two
    const float cs = a.scale * unit;

    // ---- one tile's raw rows on their way ----
    vlt5_u32x4_t kr[KP];
    uint32_t vr[8][VW];
    float scl = 0.f;
    // rows of a 16-key group are in one page; `row` = first cache row of the group, or -1
    auto group_row = [&](int t) -> long long {
        const int pg = t < hi ? paged_page(a.s, b, t) : -1;
        return pg < 0 ? -1 : (long long)((((size_t)pg * a.Hkv + hk) << a.s.page_shift) + (t & ((1 << a.s.page_shift) - 1)));
    };
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int key = __builtin_amdgcn_readfirstlane((i * 256 + w * 64) / KCH) + lane / KCH;      // 64 / KCH keys a wave: 4 .. 16
            const long long g0 = group_row(t0 + __builtin_amdgcn_readfirstlane((i * 256 + w * 64) / KCH / 16 * 16));
            kr[i] = *reinterpret_cast<const vlt5_u32x4_t*>(a.k + (size_t)(max(g0, 0LL) + (key & 15)) * ROWB + (lane % KCH) * 16);
        }
        const long long g0 = group_row(t0 + w * 16);
        const unsigned char* vp = a.v + (size_t)max(g0, 0LL) * ROWB + r32 * (NT * BY);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned char* p = vp + (size_t)((e >> 2) * 8 + h * 4 + (e & 3)) * ROWB;
            if constexpr (NT * BY == 8) { const uint2 u = *reinterpret_cast<const uint2*>(p); vr[e][0] = u.x; vr[e][1] = u.y; }
            else if constexpr (NT * BY == 4) vr[e][0] = *reinterpret_cast<const uint32_t*>(p);
            else vr[e][0] = *reinterpret_cast<const uint16_t*>(p);
        }
        if constexpr (KvType<T>::SCALED) {
            if (w < 2) {                                                                // wave 0: key scales, wave 1: value scales
                const int pg = t0 + lane < hi ? paged_page(a.s, b, t0 + lane) : -1;
                const size_t at = (((size_t)max(pg, 0) * a.Hkv + hk) << a.s.page_shift) + ((t0 + lane) & ((1 << a.s.page_shift) - 1));
                scl = (w ? a.vs : a.ks)[at];
                if (w && (pg < 0 || t0 + lane >= sq.len)) scl = 0.f;
            }
        }
        // what lies behind the last key or in a page that is not there may hold anything, NaN too
        if (t0 + w * 16 + 16 > sq.len || g0 < 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (g0 < 0 || t0 + w * 16 + (e >> 2) * 8 + h * 4 + (e & 3) >= sq.len)
#pragma unroll
                    for (int i = 0; i < VW; ++i) vr[e][i] = 0;
        }
    };
    auto stage = [&](char* buf) {
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            char* p = buf + ((i * 256 + w * 64) / KCH + lane / KCH) * KROW + (lane % KCH) * (16 / BY * 2);
            if constexpr (T == VLT5_KV_BF16) {
                *reinterpret_cast<vlt5_u32x4_t*>(p) = kr[i];
            } else {
                const uint2 c0 = codes_to_bf16<T>(kr[i].x), c1 = codes_to_bf16<T>(kr[i].y), c2 = codes_to_bf16<T>(kr[i].z), c3 = codes_to_bf16<T>(kr[i].w);
                *reinterpret_cast<uint4*>(p) = make_uint4(c0.x, c0.y, c1.x, c1.y);
                *reinterpret_cast<uint4*>(p + 16) = make_uint4(c2.x, c2.y, c3.x, c3.y);
            }
        }
        char* v = buf + KBYTES;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            uint32_t q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t x = vr[2 * e][j * BY / 4], y = vr[2 * e + 1][j * BY / 4];
                if constexpr (T == VLT5_KV_BF16) q[e] = __builtin_amdgcn_perm(y, x, j & 1 ? 0x07060302u : 0x05040100u);
                else if constexpr (T == VLT5_KV_INT8) q[e] = pack_bf16x2(sbyte(x, j), sbyte(y, j));
                else q[e] = cvt_fp8_pair(__builtin_amdgcn_perm(y, x, j & 2 ? 0x07030602u : 0x05010400u), j & 1);
            }
            *reinterpret_cast<uint4*>(v + ((w * NT + j) * 64 + lane) * 16) = make_uint4(q[0], q[1], q[2], q[3]);
        }
        if constexpr (KvType<T>::SCALED)
            if (w < 2) reinterpret_cast<float*>(v + VBYTES)[w * 64 + lane] = scl;
    };

    f32x16_t o[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[j][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    if (lo < hi) {
        fetch(lo);
        stage(smem);
    }
    __syncthreads();
    int cur = 0;
    for (int t0 = lo; t0 < hi; t0 += 64, cur ^= 1) {
        const char* buf = smem + cur * BUF;
        const bool more = t0 + 64 < hi;
        if (more) fetch(t0 + 64);
        if (t0 < wLmax) {
            f32x16_t s[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[i][e] = 0.f;
#pragma unroll
                for (int k = 0; k < NKS; ++k)
                    s[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(buf + (i * 32 + r32) * KROW + (k * 16 + h * 8) * 2), fq[k], s[i], 0, 0, 0);
            }
            // register e of tile i: key t0 + i * 32 + 8 * (e / 4) + 4 * h + e % 4
            bool there = true;
            if (t0 + 64 > wLmin) there = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) there = there && group_row(t0 + i * 16) >= 0;
            const float* ks = reinterpret_cast<const float*>(buf + KBYTES + VBYTES);
            float c = cs;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float4 k4 = make_float4(1.f, 1.f, 1.f, 1.f);
                    if constexpr (KvType<T>::SCALED) k4 = *reinterpret_cast<const float4*>(ks + i * 32 + q * 8 + h * 4);
                    const float kk[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = s[i][q * 4 + e] * (KvType<T>::SCALED ? kk[e] * c : c);
                        const int t = t0 + i * 32 + q * 8 + h * 4 + e;
                        if constexpr (BIAS) v += bias[min(max(pos - t, 0), a.nd - 1)];
                        s[i][q * 4 + e] = v;
                    }
                }
            if (!there) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const bool page = group_row(t0 + i * 32 + q / 2 * 16) >= 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[i][q * 4 + e] = page && t0 + i * 32 + q * 8 + h * 4 + e < L ? s[i][q * 4 + e] : -INFINITY;
                    }
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, s[i][e]);
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__any(top > m + 8.f * unit / LOG2E)) {
                const float mn = fmaxf(m, top), ms = mn == -INFINITY ? 0.f : mn;
                const float fix = exp2_hw((m - ms) * (BIAS ? LOG2E : 1.f));
                m = mn;
                l *= fix;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[j][e] *= fix;
            }
            const float ms = m == -INFINITY ? 0.f : m;
            bf16x8_t fp[4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int g2 = 0; g2 < 2; ++g2) {
                    uint32_t pk[4];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float4 v4 = make_float4(1.f, 1.f, 1.f, 1.f);
                        if constexpr (KvType<T>::SCALED) v4 = *reinterpret_cast<const float4*>(ks + 64 + i * 32 + (g2 * 2 + q) * 8 + h * 4);
                        const float vv[4] = {v4.x, v4.y, v4.z, v4.w};
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float d = s[i][(g2 * 2 + q) * 4 + e] - ms;
                            const float pe = exp2_hw(BIAS ? d * LOG2E : d);
                            l += pe;
                            x[e] = KvType<T>::SCALED ? pe * vv[e] : pe;
                        }
                        pk[q * 2] = pack_bf16x2(x[0], x[1]);
                        pk[q * 2 + 1] = pack_bf16x2(x[2], x[3]);
                    }
                    fp[i * 2 + g2] = __builtin_bit_cast(bf16x8_t, make_uint4(pk[0], pk[1], pk[2], pk[3]));
                }
            const char* v = buf + KBYTES;
#pragma unroll
            for (int g2 = 0; g2 < 4; ++g2)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    o[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(v + ((g2 * NT + j) * 64 + lane) * 16), fp[g2], o[j], 0, 0, 0);
        }
        if (more) stage(smem + (cur ^ 1) * BUF);
        __syncthreads();
    }
    l += __shfl_xor(l, 32, 64);
    if (wr0 + r32 >= rows) return;
    const float mnat = BIAS ? m : m / LOG2E;
    const size_t row = (size_t)(sq.q0 + tok) * a.H + hq;
    if (a.splits == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        bf16_t* dst = a.out + (size_t)(sq.q0 + tok) * a.o_st + hq * DK;
#pragma unroll
        for (int q = 0; q < 4; ++q) {                                                   // rows m = 8 q + 4 h .. + 3 of the NT tiles: 4 NT neighbouring d
            uint32_t u[2 * NT];
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) u[i] = pack_bf16x2(o[2 * i % NT][q * 4 + 2 * i / NT] * inv, o[(2 * i + 1) % NT][q * 4 + (2 * i + 1) / NT] * inv);
#pragma unroll
            for (int i = 0; i < NT / 2; ++i) *reinterpret_cast<uint4*>(dst + NT * (8 * q + 4 * h) + i * 8) = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
        }
        if (a.lse && h == 0) a.lse[row] = l == 0.f ? -INFINITY : mnat + logf(l);
    } else {
        const size_t at = (size_t)sp * a.s.n_tok * a.H + row;
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < NT; ++i)
                *reinterpret_cast<float4*>(a.part_o + at * DK + NT * (8 * q + 4 * h) + 4 * i) =
                    make_float4(o[4 * i % NT][q * 4 + 4 * i / NT], o[(4 * i + 1) % NT][q * 4 + (4 * i + 1) / NT], o[(4 * i + 2) % NT][q * 4 + (4 * i + 2) / NT],
                                o[(4 * i + 3) % NT][q * 4 + (4 * i + 3) / NT]);
        if (h == 0) { a.part_ml[at * 2] = mnat; a.part_ml[at * 2 + 1] = l; }
    }
}

// joins the splits of a row, in their order
template <int DK>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttnArgs a) {
    int id = blockIdx.x;
    const int rt = id % a.join_tiles; id /= a.join_tiles;
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

// The plan of a call, from what the host knows.  Up to 64 rows (tokens x heads of a group) go through the first kernel, more share their keys
// through LDS.  Keys are shared out until the chip is full (1024 waves' worth of small workgroups, 512 large ones), no share below 512 keys.
template <int T, int DK, bool BIAS>
int chunk_launch(const PagedAttnArgs& a, unsigned blocks, hipStream_t st) {
    static std::atomic<unsigned long long> done{0};
    constexpr int bytes = 2 * (64 * (DK * 2 + 16) + 4 * (DK / 32) * 1024 + 512);
    const int rc = vlt5_lds_optin((const void*)paged_chunk_kernel<T, DK, BIAS>, bytes, done);
    if (rc) return rc;
    hipLaunchKernelGGL((paged_chunk_kernel<T, DK, BIAS>), dim3(blocks), dim3(256), bytes, st, a);
    return VLT5_OK;
}
struct PagedPlan { int chunk, row_tiles, splits; };
PagedPlan paged_plan(const vlt5_paged_attn_desc* d, const PagedSeqs& s) {
    const int g = d->H / d->kv.n_kv_heads;
    const long long rows = (long long)s.max_q * g;
    PagedPlan p;
    p.chunk = rows > 64;
    const int per = p.chunk ? 128 : 16;
    p.row_tiles = (int)((rows + per - 1) / per);
    const long long most_kv = d->max_kv > 0 ? d->max_kv : (long long)d->seqs.max_pages * d->kv.page_size;
    const long long tiles = (long long)s.B * d->kv.n_kv_heads * p.row_tiles;
    long long sp = ((p.chunk ? 512 : 1024) + tiles - 1) / tiles;
    sp = sp < most_kv / 512 ? sp : most_kv / 512;
    p.splits = (int)(sp < 1 ? 1 : (sp > 64 ? 64 : sp));
    return p;
}

}  // namespace

int vlt5_paged_check(const vlt5_paged_kv* c, const vlt5_paged_seqs* q);
PagedSeqs vlt5_paged_seqs_of(const vlt5_paged_kv* c, const vlt5_paged_seqs* q);

extern "C" long long vlt5_paged_attn_workspace_bytes(const vlt5_paged_attn_desc* d) {
    if (!d || vlt5_paged_check(&d->kv, &d->seqs) || d->H <= 0 || d->H % d->kv.n_kv_heads) return -1;
    const PagedSeqs s = vlt5_paged_seqs_of(&d->kv, &d->seqs);
    const int sp = paged_plan(d, s).splits;
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
    const PagedPlan plan = paged_plan(d, a.s);
    a.row_tiles = plan.row_tiles; a.splits = plan.splits; a.join_tiles = (int)(((long long)a.s.max_q * a.g + 15) / 16);
    const long long rows = (long long)a.s.n_tok * a.H;
    if (a.splits > 1) {
        if (!d->workspace || d->workspace_bytes < (long long)a.splits * rows * (c.d_kv + 2) * 4) return VLT5_ERR_ARG;
        a.part_o = (float*)d->workspace;
        a.part_ml = a.part_o + (size_t)a.splits * rows * c.d_kv;
    } else {
        a.part_o = a.part_ml = nullptr;
    }
    const long long tiles = (long long)a.s.B * a.Hkv * a.row_tiles;
    const long long joins = (long long)a.s.B * a.Hkv * a.join_tiles;
    if (tiles * a.splits > 0x7fffffffLL || joins > 0x7fffffffLL) return VLT5_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    int lrc = VLT5_OK;
#define PA(T, D) do { if (plan.chunk) lrc = a.bias ? chunk_launch<T, D, true>(a, (unsigned)(tiles * a.splits), st) : chunk_launch<T, D, false>(a, (unsigned)(tiles * a.splits), st); \
                      else hipLaunchKernelGGL((paged_attn_kernel<T, D, 4>), dim3((unsigned)(tiles * a.splits)), dim3(256), 0, st, a); } while (0)
    if (c.d_kv == 64) {
        if (c.type == VLT5_KV_BF16) PA(VLT5_KV_BF16, 64); else if (c.type == VLT5_KV_INT8) PA(VLT5_KV_INT8, 64); else PA(VLT5_KV_FP8, 64);
    } else {
        if (c.type == VLT5_KV_BF16) PA(VLT5_KV_BF16, 128); else if (c.type == VLT5_KV_INT8) PA(VLT5_KV_INT8, 128); else PA(VLT5_KV_FP8, 128);
    }
#undef PA
    if (lrc) return lrc;
    LAUNCH_CHECK();
    if (a.splits > 1) {
        if (c.d_kv == 64) hipLaunchKernelGGL(paged_join_kernel<64>, dim3((unsigned)joins), dim3(256), 0, st, a);
        else hipLaunchKernelGGL(paged_join_kernel<128>, dim3((unsigned)joins), dim3(256), 0, st, a);
        LAUNCH_CHECK();
    }
    return VLT5_OK;
}
