// Attention of the newest tokens of every sequence over its paged cache: softmax(scale * q K^T + bias) V, single tokens and chunks.
//
// The query rows of one (sequence, kv head) are the tokens times the query heads that share the kv head.  Few rows (paged_attn_kernel): sixteen
// a tile, every wave for itself, everything in registers.  Many rows (paged_chunk_kernel): 128 a workgroup, keys and values converted to bf16
// once and shared through LDS.  In both, with the running maximum and sum of the softmax in f32:
//   scores  S^T[key, row] = mfma(A = keys, B = query rows): a lane ends up with runs of four consecutive keys of ONE row;
//   output  O^T[d, row] += mfma(A = V^T, B = P^T): the keys of one instruction may be taken in any order as long as both operands agree, so
//           the eight keys of a lane's B operand are simply ones it has scores of -- no exchange between lanes -- and the A operand is built
//           from the same eight rows of V, a few neighbouring values of each: the conversion to bf16 pairs them by key, which IS the
//           transposition.
// 8-bit codes are exact in bf16; the scale of a key multiplies its score, the scale of a value its probability (in f32, before the one
// rounding of the probabilities to bf16, which with the output's own is all the rounding there is below 32 bits).
//
// Single tokens are bound by the bytes of the cache: 32 x 8192 - 16384 keys, 8 kv heads of 128, e4m3: 148 - 151 us = 5.5 TB/s (of 6.2 that a kernel
// which does nothing but read reaches); in bf16 at 16384 each 372 us = 5.8.  1 x 131071, int8: 59 - 63 us a call = 4.4 - 4.7 TB/s, 4.7 of them to join
// its 64 shares (48 where the same cache is read again and again: the last-level cache holds a part of it); in bf16 105 us.  Long chunks are
// bound by the matrix and vector units together (42 % and 41 % busy at the 1.8 GHz such a load runs at): 2048 tokens over 16384 keys, 32 heads of
// 128, 545 - 590 us in bf16 = 875 - 945 TFLOP/s (the first dozen launches of a process 620 - 670), 577 in e4m3, 603 in int8.
#include "paged.h"
#include "rows.h"

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

// Makes the compiler wait for a loaded operand HERE: left to its first use inside a loop, the wait would be repeated in every pass and hold up
// the loads of the pass after (they are counted in order).
template <class V>
__device__ __forceinline__ void arrived(V& f) { asm volatile("" : "+v"(f)); }

// The bias of a row tile's heads is read from LDS where it fits this many entries: a gather from memory would wait for the keys requested before it.
constexpr int BIAS_LDS = 1024;

constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

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

// Values that are not finite.  A masked probability of 0 times such a value is not 0, so where some rows of a workgroup see a key that others do not
// (causal, the last keys), they are taken out of V on its way into the product (bf16 and e4m3; an int8 value is always finite), and the first
// position of +inf and of -inf is kept for each d (a NaN counts as both): with the mask a row sees that position or it sees none of them, so the
// row's output gains +inf, -inf or both, which is NaN, at the end.  Elsewhere every row sees the key and the product gives what it gives.
// It costs a look at the values of the last tiles and a barrier: 8 x 16 tokens over 500 bf16 keys, 12 heads of 64, 8.1 -> 8.8 us, 8 x 5 over 3000, 32 / 8
// of 128, 32.4 -> 34.9, 45 x 79 over 79 11.6 -> 12.0, 1 x 1000 over 8000 98.1 -> 98.3.
struct OddValues {                                     // in LDS: first position of +inf by d, of -inf by d (or MOST), are there any?
    int* at; int dk;
    static constexpr int MOST = 0x7fffffff;
    __device__ __forceinline__ void clear(int tid, int threads) const {
        for (int i = tid; i < 2 * dk + 1; i += threads) at[i] = i < 2 * dk ? MOST : 0;
    }
    __device__ __forceinline__ bool any() const { return __builtin_amdgcn_readfirstlane(at[2 * dk]); }
    __device__ __forceinline__ float add(int d, int len) const { return (at[d] < len ? INFINITY : 0.f) + (at[dk + d] < len ? -INFINITY : 0.f); }
};
template <int T>
__device__ __forceinline__ bool odd_values(uint32_t w) {   // any in a raw dword?
    if constexpr (T == VLT5_KV_BF16) return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    else if constexpr (T == VLT5_KV_FP8) return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    else return false;
}
// takes them out of a raw dword that holds d, d + 1, .. of the key at `pos`
template <int T>
__device__ __forceinline__ void take_odd(uint32_t& w, const OddValues& o, int d, int pos) {
    constexpr int BITS = 8 * KvType<T>::BYTES;
    for (int i = 0; i < 32 / BITS; ++i) {
        const uint32_t x = w >> (i * BITS) & (0xffffffffu >> (32 - BITS)), mag = T == VLT5_KV_BF16 ? x & 0x7fffu : x & 0x7fu;
        if (mag < (T == VLT5_KV_BF16 ? 0x7f80u : 0x7fu)) continue;
        const bool nan = T == VLT5_KV_FP8 || mag > 0x7f80u;
        if (nan || x == mag) atomicMin(o.at + d + i, pos);
        if (nan || x != mag) atomicMin(o.at + o.dk + d + i, pos);
        o.at[2 * o.dk] = 1;
        w &= ~((0xffffffffu >> (32 - BITS)) << (i * BITS));
    }
}

// The raw rows of 32 keys, as one lane holds them: for the scores keys 16 i + lane % 16 (16-byte pieces of the row), for the output the rows
// 16 i + 4 * (lane / 16) + 0 .. 3, DK / 16 values of each.
template <int T, int DK>
struct KeyStep {
    static constexpr int KP = DK * KvType<T>::BYTES / 64;
    vlt5_u32x4_t k[2][KP];
    VRow<T, DK> v[2][4];
    float4 ks[2], vs[2];
    __device__ __forceinline__ void load(const PagedAttnArgs& a, int hk, const int (&page)[2], int t, int r16, int kq) {
        constexpr int ROWB = DK * KvType<T>::BYTES;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const size_t base = (((size_t)max(page[i], 0) * a.Hkv + hk) << a.s.page_shift) + ((t + i * 16) & ((1 << a.s.page_shift) - 1));
            const unsigned char* kp = a.k + (base + r16) * ROWB + kq * 16;
#pragma unroll
            for (int c = 0; c < KP; ++c) k[i][c] = *reinterpret_cast<const vlt5_u32x4_t*>(kp + c * 64);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = load_vrow<T, DK>(a.v + (base + kq * 4 + e) * ROWB + r16 * (ROWB / 16));
            if constexpr (KvType<T>::SCALED) {
                ks[i] = *reinterpret_cast<const float4*>(a.ks + base + kq * 4);
                vs[i] = *reinterpret_cast<const float4*>(a.vs + base + kq * 4);
            }
        }
    }
};

// NW waves share the keys of 16 R rows in steps of 32, the next step's rows on their way while one is used; the page ids of a wave's next 32 steps
// come with one load, two to a step.  The R row tiles use the same operands of K and V: a key is read and converted once for all of them.
// ODD: a causal call of several tokens a sequence, whose last keys some of its rows do not see (single tokens see all: without the code for it three
// waves of the 64-wide form fit a SIMD, with it two).
template <int T, int DK, int NW, int R, bool ODD>
__global__ __launch_bounds__(NW * 64, R * DK > 128 ? 1 : 2) void paged_attn_kernel(const PagedAttnArgs a) {
    constexpr int NF = DK / 32, ND = DK / 16;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, kq = lane >> 4;
    int id = blockIdx.x;
    const int sp = id % a.splits; id /= a.splits;
    const int rt = id % a.row_tiles; id /= a.row_tiles;
    const int hk = id % a.Hkv, b = id / a.Hkv;
    const PagedSeq sq = paged_seq(a.s, b);
    const int rows = min(sq.nq, a.s.max_q) * a.g, r0 = rt * 16 * R;
    if (r0 >= rows) return;
    const int p0 = sq.len - sq.nq;
    const int first = p0 + r0 / a.g, last = p0 + min(r0 + 16 * R - 1, rows - 1) / a.g;
    const int Lmin = a.causal ? first + 1 : sq.len, Lmax = max(a.causal ? last + 1 : sq.len, 0);
    const int per = ((Lmax + a.splits - 1) / a.splits + 32 * NW - 1) / (32 * NW) * (32 * NW);
    const int lo = min(sp * per, Lmax), hi = min(lo + per, Lmax);

    // what the first step needs is requested in the order it is waited for: page ids, query rows, bias, (keys and values below)
    const int steps = hi > lo ? (hi - lo + 31) / 32 : 0, mine = steps > w ? (steps - w + NW - 1) / NW : 0;
    auto at = [&](int i) { return lo + (i * NW + w) * 32; };
    int ids = -1;                                                                  // lane j: page of the 16 keys j & 1 of step (i & ~31) + j / 2
    auto load_ids = [&](int i) {
        const int t = at(i + (lane >> 1)) + (lane & 1) * 16;
        ids = i + (lane >> 1) < mine && t < hi ? a.s.table[(size_t)b * a.s.max_pages + (t >> a.s.page_shift)] : -1;
    };
    auto settle_ids = [&] {
        arrived(ids);
        if ((unsigned)ids >= (unsigned)a.s.n_pages) ids = -1;
    };
    if (mine) load_ids(0);
    int pos[R], L[R], head[R];                                                     // position of this lane's row (negative: more new tokens than keys), keys it sees, its head
    bf16x8_t fq[R][NF];                                                            // d in the order of the keys' 16-byte pieces
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = min(r0 + i * 16 + r16, rows - 1), tok = r / a.g;
        head[i] = r % a.g;
        pos[i] = p0 + tok;
        L[i] = a.causal ? min(pos[i] + 1, sq.len) : sq.len;
        const bf16_t* qrow = a.q + (size_t)(sq.q0 + tok) * a.q_st + (hk * a.g + head[i]) * DK;
#pragma unroll
        for (int f = 0; f < NF; ++f) fq[i][f] = *reinterpret_cast<const bf16x8_t*>(qrow + (T == VLT5_KV_BF16 ? f * 32 + kq * 8 : (f >> 1) * 64 + kq * 16 + (f & 1) * 8));
    }
    __shared__ int first_odd[ODD ? 2 * DK + 1 : 1];
    const OddValues odd = {first_odd, DK};
    const bool track = ODD && first != last;
    if (track) odd.clear(threadIdx.x, NW * 64);
    __shared__ float sb[BIAS_LDS];
    const bool near_lds = a.bias && a.g * a.nd <= BIAS_LDS;
    const float* bias = a.bias ? a.bias + (size_t)hk * a.g * a.nd : nullptr;
    float table[2];
    if (near_lds)
#pragma unroll
        for (int i = 0; i < 2; ++i) table[i] = bias[min((int)threadIdx.x + i * NW * 64, a.g * a.nd - 1)];
    float bias_far[R];
#pragma unroll
    for (int i = 0; i < R; ++i) bias_far[i] = bias ? bias[head[i] * a.nd + a.nd - 1] : 0.f;
    if (mine) settle_ids();
    // scores and their maximum are kept as q k (times the key's scale), with a bias as scale * q k + bias; `unit` makes powers of two of them
    const float unit = bias ? LOG2E : a.scale * LOG2E, lag = fminf(8.f / unit, 1e38f);

    f32x4_t o[R][ND];
    float m[R], l[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int j = 0; j < ND; ++j) o[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    int pg[2][2];
    KeyStep<T, DK> st[2];
    auto load = [&](int i, int buf) {
        pg[buf][0] = __builtin_amdgcn_readlane(ids, (i & 31) * 2);
        pg[buf][1] = __builtin_amdgcn_readlane(ids, (i & 31) * 2 + 1);
        st[buf].load(a, hk, pg[buf], at(i), r16, kq);
    };
    auto use = [&](int step, int buf) {
        KeyStep<T, DK>& x = st[buf];
        const int t0 = at(step);
        f32x4_t sc[R][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int q = 0; q < R; ++q) sc[q][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                bf16x8_t fk;
                if constexpr (T == VLT5_KV_BF16) fk = __builtin_bit_cast(bf16x8_t, x.k[i][f]);
                else {
                    const uint2 c0 = codes_to_bf16<T>(x.k[i][f >> 1][(f & 1) * 2]), c1 = codes_to_bf16<T>(x.k[i][f >> 1][(f & 1) * 2 + 1]);
                    fk = __builtin_bit_cast(bf16x8_t, make_uint4(c0.x, c0.y, c1.x, c1.y));
                }
#pragma unroll
                for (int q = 0; q < R; ++q) sc[q][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fk, fq[q][f], sc[q][i], 0, 0, 0);
            }
        }
        const bool whole = t0 + 32 <= min(Lmin, hi) && pg[buf][0] >= 0 && pg[buf][1] >= 0;
        bf16x8_t fp[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            float p[2][4], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float kk[4] = {1.f, 1.f, 1.f, 1.f};
                if constexpr (KvType<T>::SCALED) { kk[0] = x.ks[i].x; kk[1] = x.ks[i].y; kk[2] = x.ks[i].z; kk[3] = x.ks[i].w; }
#pragma unroll
                for (int e = 0; e < 4; ++e) p[i][e] = sc[q][i][e] * kk[e];
            }
            if (bias) {
                if (first - (t0 + 31) >= a.nd - 1) {                               // every key further than the table reaches
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[i][e] = fmaf(p[i][e], a.scale, bias_far[q]);
                } else if (near_lds) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            p[i][e] = fmaf(p[i][e], a.scale, sb[head[q] * a.nd + min(max(pos[q] - (t0 + i * 16 + kq * 4 + e), 0), a.nd - 1)]);
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            p[i][e] = fmaf(p[i][e], a.scale, bias[head[q] * a.nd + min(max(pos[q] - (t0 + i * 16 + kq * 4 + e), 0), a.nd - 1)]);
                }
            }
            if (!whole) {
                asm volatile("");                                                  // (a branch, not selects in every step)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[i][e] = pg[buf][i] >= 0 && t0 + i * 16 + kq * 4 + e < L[q] ? p[i][e] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, p[i][e]);
            // the running maximum moves only when a new one is more than 2^8 away: until then probabilities up to 256 do no harm (f32 sums, bf16
            // relative to the value), and neither the exchange between the row's four lanes nor the rescaling is needed
            if (__any(top > m[q] + lag)) {
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float mn = fmaxf(m[q], top), ms = mn == -INFINITY ? 0.f : mn;    // a row that has seen no key yet stays at -inf, sum 0
                const float fix = exp2_hw((m[q] - ms) * unit);
                m[q] = mn;
                l[q] *= fix;
#pragma unroll
                for (int j = 0; j < ND; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[q][j][e] *= fix;
            }
            const float ms = m[q] == -INFINITY ? 0.f : m[q];
            uint32_t pb[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float vv[4] = {1.f, 1.f, 1.f, 1.f}, y[4];
                if constexpr (KvType<T>::SCALED) { vv[0] = x.vs[i].x; vv[1] = x.vs[i].y; vv[2] = x.vs[i].z; vv[3] = x.vs[i].w; }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float pe = exp2_hw((p[i][e] - ms) * unit);
                    l[q] += pe;
                    y[e] = pe * vv[e];
                }
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = pg[buf][i] >= 0 && t0 + i * 16 + kq * 4 + e < L[q] ? y[e] : 0.f;
                }
                pb[i][0] = pack_bf16x2(y[0], y[1]);
                pb[i][1] = pack_bf16x2(y[2], y[3]);
            }
            fp[q] = __builtin_bit_cast(bf16x8_t, make_uint4(pb[0][0], pb[0][1], pb[1][0], pb[1][1]));
        }
        if (!whole) {                                                              // what lies behind the last key that a row sees may hold anything, NaN too
            asm volatile("");
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!(pg[buf][i] >= 0 && t0 + i * 16 + kq * 4 + e < Lmax)) x.v[i][e] = VRow<T, DK>{};
            if (track) {
                bool any = false;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (uint32_t v : x.v[i][e].w) any |= odd_values<T>(v);
                if (__builtin_expect(any, 0)) {
                    int me = threadIdx.x;
                    asm volatile("" : "+v"(me));                                   // (what follows is formed here: kept since the start it would spill)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int n = 0; n < (int)(sizeof x.v[i][e].w / 4); ++n)
                                take_odd<T>(x.v[i][e].w[n], odd, me % 16 * ND + n * 4 / KvType<T>::BYTES, t0 + i * 16 + me / 16 % 4 * 4 + e);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < ND; ++j) {
            const uint4 fv = make_uint4(vpair<T, DK>(x.v[0][0], x.v[0][1], j), vpair<T, DK>(x.v[0][2], x.v[0][3], j), vpair<T, DK>(x.v[1][0], x.v[1][1], j),
                                        vpair<T, DK>(x.v[1][2], x.v[1][3], j));
#pragma unroll
            for (int q = 0; q < R; ++q) o[q][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, fv), fp[q], o[q][j], 0, 0, 0);
        }
    };
    if (mine) load(0, 0);
#pragma unroll
    for (int q = 0; q < R; ++q) {
#pragma unroll
        for (int f = 0; f < NF; ++f) arrived(fq[q][f]);
        arrived(bias_far[q]);
    }
    if (near_lds) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if ((int)threadIdx.x + k * NW * 64 < a.g * a.nd) sb[threadIdx.x + k * NW * 64] = table[k];
        for (int k = threadIdx.x + 2 * NW * 64; k < a.g * a.nd; k += NW * 64) sb[k] = bias[k];
    }
    if (near_lds || track) __syncthreads();
    int i = 0;
    for (; i + 2 < mine; i += 2) {                                                 // (every load unconditional, or the waits could not be counted)
        load(i + 1, 1);                                                            // (i is even: never the first of 32 steps)
        use(i, 0);
        if (((i + 2) & 31) == 0) {
            load_ids(i + 2);
            settle_ids();
        }
        load(i + 2, 0);
        use(i + 1, 1);
    }
    if (i + 1 < mine) {
        load(i + 1, 1);
        use(i, 0);
        use(i + 1, 1);
    } else if (i < mine) {
        use(i, 0);
    }

    // ---- the waves' shares of the keys meet in LDS, always in the order of the waves, one row tile after the other ----
    __shared__ float so[NW][16][DK + 4];
    __shared__ float sm[NW][16], sl[NW][16];
#pragma unroll
    for (int q = 0; q < R; ++q) {
        l[q] += __shfl_xor(l[q], 16, 64);
        l[q] += __shfl_xor(l[q], 32, 64);
        if (q) __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < ND; ++j) so[w][r16][(kq * 4 + e) * ND + j] = o[q][j][e];      // row of the A operand (kq * 4 + e) stands for d = that * ND + j
        if (lane < 16) { sm[w][lane] = bias ? m[q] : m[q] * a.scale; sl[w][lane] = l[q]; }
        __syncthreads();
        for (int k = threadIdx.x; k < 16 * (DK / 4); k += NW * 64) {
            const int rr = k / (DK / 4), d = k % (DK / 4) * 4, r = r0 + q * 16 + rr;
            if (r >= rows) continue;
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
            if (track && odd.any()) {
                const int len = min(p0 + r / a.g + 1, sq.len);
                acc.x += odd.add(d, len); acc.y += odd.add(d + 1, len); acc.z += odd.add(d + 2, len); acc.w += odd.add(d + 3, len);
            }
            const int hh = hk * a.g + r % a.g;
            const size_t token = (size_t)(sq.q0 + r / a.g);
            if (a.splits == 1) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                *reinterpret_cast<uint2*>(a.out + token * a.o_st + hh * DK + d) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
                if (a.lse && d == 0) a.lse[token * a.H + hh] = sum == 0.f ? -INFINITY : mx + logf(sum);
            } else {
                const size_t row = ((size_t)sp * a.s.n_tok + token) * a.H + hh;
                *reinterpret_cast<float4*>(a.part_o + row * DK + d) = acc;
                if (d == 0) { a.part_ml[row * 2] = mx; a.part_ml[row * 2 + 1] = sum; }
            }
        }
    }
}

// Room for the chunk kernel's bias tables, one per head of the group: distances from -PAD on (keys past a row's own, masked) to PAD past the last
// entry, so that a tile's 32 entries of a lane lie at fixed places from one address, with no index arithmetic and few registers: the 64-wide form
// leaves a CU three workgroups instead of two (45 x 79 tokens over 79 keys, 12 heads, int8, 128 distances: 13.1 -> 10.8 us, 9.5 without a bias; all of
// them 79 long 14.0, 12.3 without; two to six registers that only the end needs are put away in front of the loop for it).  Larger tables, as of seven
// heads a group with 128 distances, are read from memory, which costs no more where heads share: 8 x 200 over 712, 32 / 4 heads of 64, int8, 64 distances (LDS) 34.0 us, 65 (memory) 32.0,
// 128 36.2, none 28.4; with a head a group 1856 distances 22.5 and 1857 25.3.
constexpr int CHUNK_BIAS_LDS = 2048, PAD = 96;

// ---- chunks: many rows share the keys ------------------------------------------------------------------------------------------------
// 128 query rows a workgroup, 32 of them a wave; tiles of 64 keys and values are converted to bf16 ONCE per workgroup on their way into LDS
// (two buffers: the next tile's loads are in flight while one is used), the same two products as above on 32 x 32 x 16 instructions.
//   K in LDS: rows of d_kv values + 16 bytes, so that 16 rows of an operand start in 16 bank groups;
//   V in LDS: in the order the operand wants it, [16 keys][d % NT][lane] pieces of eight keys of one d -- the thread that loaded d_kv / 32
//   neighbouring values of eight rows pairs them by key; d = NT * m + j for row m of operand tile j makes its stores and the reads consecutive.
// The running maximum moves only when a row's new one is more than 2^8 away: until then probabilities up to 256 are exact enough in every
// type they pass through (f32 sums, bf16 relative to the value), and the output's 16 * NT registers are left alone.
typedef __attribute__((ext_vector_type(16))) float f32x16_t;

template <int T, int DK, bool BIAS, int KS>
__global__ __launch_bounds__(256 * KS, DK == 64 && KS == 1 ? 3 : 2) void paged_chunk_kernel(const PagedAttnArgs a) {
    constexpr int NT = DK / 32, NKS = DK / 16, BY = KvType<T>::BYTES, ROWB = DK * BY;
    constexpr int KROW = DK * 2 + 16, KBYTES = 64 * KROW, VBYTES = 4 * NT * 1024, BUF = KBYTES + VBYTES + 512;
    constexpr int KCH = ROWB / 16, KP = 64 * KCH / 256;                                 // 16-byte pieces of a key row; pieces of a thread
    constexpr int VW = (NT * BY + 3) / 4;                                               // dwords of a thread's share of a value row
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r32 = lane & 31, h = lane >> 5;
    const int w4 = w & 3, half = w >> 2;                                                // wave of its half, half
    const int pairs = a.s.B * a.Hkv;
    const int pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
    const int sp = rest % a.splits, rt = a.row_tiles - 1 - rest / a.splits;             // the last rows see the most keys: they start first
    const int hk = pair % a.Hkv, b = pair / a.Hkv;
    const PagedSeq sq = paged_seq(a.s, b);
    const int rows = min(sq.nq, a.s.max_q) * a.g;
    if (rt * 128 >= rows) return;
    const int wr0 = rt * 128 + w4 * 32;                                                 // first row of the wave
    const int r = min(wr0 + r32, rows - 1);
    const int tok = r / a.g, hq = hk * a.g + r % a.g;
    const int p0 = sq.len - sq.nq;
    const int L = a.causal ? p0 + tok + 1 : sq.len;                                     // keys of this lane's row (with a bias its position is L - 1)
    const int Lmax = max(a.causal ? p0 + min(rt * 128 + 127, rows - 1) / a.g + 1 : sq.len, 0);
    const int wLmin = a.causal ? p0 + min(wr0, rows - 1) / a.g + 1 : sq.len;            // the wave's rows all see the keys below this ...
    const int wLmax = wr0 < rows ? (a.causal ? p0 + min(wr0 + 31, rows - 1) / a.g + 1 : sq.len) : 0;      // ... and none those from here on
    const bool track = T != VLT5_KV_INT8 && a.causal;
    const int least = p0 + rt * 128 / a.g + 1;                                          // the workgroup's rows do not all see the keys from here on
    const OddValues odd = {reinterpret_cast<int*>(smem + 2 * KS * BUF + (BIAS ? CHUNK_BIAS_LDS * 4 : 0)), DK};
    if (track) odd.clear(tid, 256 * KS);
    const int per = ((Lmax + a.splits - 1) / a.splits + 63) & ~63;
    const int lo = min(sp * per, Lmax), hi = min(lo + per, Lmax);

    // what the first tile needs is requested in the order it is waited for: page ids, query rows, bias, (keys and values below)
    // the keys of 16 are in one page; lane j: page of the j-th 16 keys of the 16 tiles from (tile & ~15) on, or -1
    int ids = -1, pg[4], pn[4];                                                         // ... and those of this tile and the next
    const int tiles = (hi - lo + 63) / 64;
    auto load_ids = [&](int tile) {
        const int t = lo + tile * 64 + lane * 16;
        ids = t < hi ? a.s.table[(size_t)b * a.s.max_pages + (t >> a.s.page_shift)] : -1;
    };
    auto settle_ids = [&] {
        arrived(ids);
        if ((unsigned)ids >= (unsigned)a.s.n_pages) ids = -1;
    };
    if (half < tiles) load_ids(0);
    bf16x8_t fq[NKS];
    const bf16_t* qrow = a.q + (size_t)(sq.q0 + tok) * a.q_st + hq * DK;
#pragma unroll
    for (int i = 0; i < NKS; ++i) fq[i] = *reinterpret_cast<const bf16x8_t*>(qrow + i * 16 + h * 8);
    const float* bias = BIAS ? a.bias + (size_t)hq * a.nd : nullptr;
    float bias_far = BIAS ? bias[a.nd - 1] : 0.f;
    float* sb = reinterpret_cast<float*>(smem + 2 * KS * BUF);
    const int span = min(a.nd, CHUNK_BIAS_LDS) + 2 * PAD, entries = a.g * span;          // (larger tables do not fit)
    const bool near_lds = BIAS && entries <= CHUNK_BIAS_LDS;
    const float* lbias = sb + (hq - hk * a.g) * span + PAD - 59;                        // (59: the largest key of a lane in a tile, not counting 4 h)
    auto entry = [&](int i) {
        int hh = 0;
        for (; i >= span; i -= span) ++hh;
        return a.bias[((size_t)hk * a.g + hh) * a.nd + min(max(i - PAD, 0), a.nd - 1)];
    };
    float table[2];
    if (near_lds)
#pragma unroll
        for (int j = 0; j < 2; ++j) table[j] = entry(min(tid + j * 256 * KS, entries - 1));
    settle_ids();
    // scores and their maximum are kept as q k (times the key's scale), with a bias as scale * q k + bias; `unit` makes powers of two of them
    const float unit = BIAS ? LOG2E : a.scale * LOG2E, lag = fminf(8.f / unit, 1e38f);

    // ---- one tile's raw rows on their way ----
    vlt5_u32x4_t kr[KP];
    uint32_t vr[8][VW];
    float ksc = 0.f, vsc = 0.f;
    bool sees = false;
    auto first_row = [&](int page, int t) { return (((size_t)max(page, 0) * a.Hkv + hk) << a.s.page_shift) + (t & ((1 << a.s.page_shift) - 1)); };
    auto fetch = [&](int tile) {
        const int t0 = lo + tile * 64;
#pragma unroll
        for (int i = 0; i < 4; ++i) pn[i] = __builtin_amdgcn_readlane(ids, (tile & 15) * 4 + i);
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            // the pieces of 64 lanes are 64 / KCH (4, 8 or 16) keys of one group of 16
            const int base = (i * 256 + w4 * 64) / KCH, grp = base >> 4;
            const int page = grp == 0 ? pn[0] : (grp == 1 ? pn[1] : (grp == 2 ? pn[2] : pn[3]));
            kr[i] = *reinterpret_cast<const vlt5_u32x4_t*>(a.k + (first_row(page, t0 + grp * 16) + ((base & 15) + lane / KCH)) * ROWB + (lane % KCH) * 16);
        }
        const int g0 = w4 == 0 ? pn[0] : (w4 == 1 ? pn[1] : (w4 == 2 ? pn[2] : pn[3]));
        const unsigned char* vp = a.v + first_row(g0, t0 + w4 * 16) * ROWB + r32 * (NT * BY);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned char* p = vp + (size_t)((e >> 2) * 8 + h * 4 + (e & 3)) * ROWB;
            if constexpr (NT * BY == 8) { const uint2 u = *reinterpret_cast<const uint2*>(p); vr[e][0] = u.x; vr[e][1] = u.y; }
            else if constexpr (NT * BY == 4) vr[e][0] = *reinterpret_cast<const uint32_t*>(p);
            else vr[e][0] = *reinterpret_cast<const uint16_t*>(p);
        }
        if constexpr (KvType<T>::SCALED) {
            if (w4 == 0) {
                const int page = lane < 16 ? pn[0] : (lane < 32 ? pn[1] : (lane < 48 ? pn[2] : pn[3]));
                const size_t at = first_row(page, t0 + lane);
                ksc = a.ks[at];
                vsc = a.vs[at];
                sees = page >= 0 && t0 + lane < sq.len;
            }
        }
        // what lies behind the last key or in a page that is not there may hold anything, NaN too
        if (t0 + w4 * 16 + 16 > sq.len || g0 < 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (g0 < 0 || t0 + w4 * 16 + (e >> 2) * 8 + h * 4 + (e & 3) >= sq.len)
#pragma unroll
                    for (int i = 0; i < VW; ++i) vr[e][i] = 0;
        }
    };
    auto stage = [&](char* buf, int tile) {
        if (track && lo + tile * 64 + 64 > least) {
            bool any = false;
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int i = 0; i < VW; ++i) any |= odd_values<T>(vr[e][i]);
            if (__builtin_expect(any, 0)) {
                int me = tid;
                asm volatile("" : "+v"(me));
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int i = 0; i < VW; ++i)
                        take_odd<T>(vr[e][i], odd, me % 32 * NT + i * 4 / BY, lo + tile * 64 + w4 * 16 + (e >> 2) * 8 + me / 32 % 2 * 4 + (e & 3));
            }
        }
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            char* p = buf + ((i * 256 + w4 * 64) / KCH + lane / KCH) * KROW + (lane % KCH) * (16 / BY * 2);
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
            *reinterpret_cast<uint4*>(v + ((w4 * NT + j) * 64 + lane) * 16) = make_uint4(q[0], q[1], q[2], q[3]);
        }
        if constexpr (KvType<T>::SCALED)
            if (w4 == 0) {
                // a value scale that is not finite moves to the key's side: a masked score is dropped, but a masked probability of 0 times it is not 0
                const bool fine = fabsf(vsc) <= 3.402823466e38f;
                reinterpret_cast<float*>(v + VBYTES)[lane] = fine ? ksc : __uint_as_float(0x7fc00000u);
                reinterpret_cast<float*>(v + VBYTES)[64 + lane] = fine && sees ? vsc : 0.f;
            }
    };

    f32x16_t o[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[j][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    char* mine = smem + half * 2 * BUF;
    if (half < tiles) fetch(half);
#pragma unroll
    for (int i = 0; i < NKS; ++i) arrived(fq[i]);
    arrived(bias_far);
    if (near_lds) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (tid + j * 256 * KS < entries) sb[tid + j * 256 * KS] = table[j];
        for (int i = tid + 512 * KS; i < entries; i += 256 * KS) sb[i] = entry(i);
    }
    if (track) __syncthreads();
    if (half < tiles) stage(mine, half);
    __syncthreads();
    for (int turn = 0; turn * KS < tiles; ++turn) {
        const int tile = turn * KS + half, t0 = lo + tile * 64, cur = turn & 1;
        const char* buf = mine + cur * BUF;
        const bool more = tile + KS < tiles;
#pragma unroll
        for (int i = 0; i < 4; ++i) pg[i] = pn[i];
        if (more) {
            if (((tile + KS) & 15) == half) {
                load_ids((tile + KS) & ~15);
                settle_ids();
            }
            fetch(tile + KS);
        }
        if (t0 < wLmax && tile < tiles) {
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
            const bool whole = t0 + 64 <= wLmin && min(min(pg[0], pg[1]), min(pg[2], pg[3])) >= 0;
            const float* ks = reinterpret_cast<const float*>(buf + KBYTES + VBYTES);
            if constexpr (KvType<T>::SCALED) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4 k4 = *reinterpret_cast<const float4*>(ks + i * 32 + q * 8 + h * 4);
                        s[i][q * 4] *= k4.x; s[i][q * 4 + 1] *= k4.y; s[i][q * 4 + 2] *= k4.z; s[i][q * 4 + 3] *= k4.w;
                    }
            }
            if constexpr (BIAS) {
                if (p0 + min(wr0, rows - 1) / a.g - (t0 + 63) >= a.nd - 1) {            // every key further than the table reaches
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[i][e] = fmaf(s[i][e], a.scale, bias_far);
                } else if (near_lds) {
                    // a row's distances here: at least -94 (its wave's last row sees the tile's first key), at most nd + 92 (the first row's nearest is in the table)
                    const float* lb = lbias + (L - 1 - t0 - h * 4);
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            s[i][e] = fmaf(s[i][e], a.scale, lb[59 - (i * 32 + e / 4 * 8 + e % 4)]);
                            if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);          // (all 32 in flight would not leave registers for the sums)
                        }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            s[i][e] = fmaf(s[i][e], a.scale, bias[min(max(L - 1 - (t0 + i * 32 + e / 4 * 8 + h * 4 + e % 4), 0), a.nd - 1)]);
                            if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                        }
                }
            }
            if (!whole) {
                asm volatile("");                                                       // (a branch, not 96 instructions of selects in every tile)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        s[i][e] = pg[i * 2 + e / 8] >= 0 && t0 + i * 32 + e / 4 * 8 + h * 4 + e % 4 < L ? s[i][e] : -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, s[i][e]);
            if (__any(top > m + lag)) {
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float mn = fmaxf(m, top), ms = mn == -INFINITY ? 0.f : mn;
                const float fix = exp2_hw((m - ms) * unit);
                m = mn;
                l *= fix;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[j][e] *= fix;
            }
            const float ms = m == -INFINITY ? 0.f : m, mu = -ms * unit;
            bf16x8_t fp[4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int g2 = 0; g2 < 2; ++g2) {
                    uint32_t pk[4];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float z = s[i][(g2 * 2 + q) * 4 + e];
                            // (with a bias not one fused operation: the type's lowest value as a mask times log2(e) would leave the range)
                            x[e] = exp2_hw(BIAS ? (z - ms) * LOG2E : fmaf(z, unit, mu));
                            l += x[e];
                        }
                        if constexpr (KvType<T>::SCALED) {
                            const float4 v4 = *reinterpret_cast<const float4*>(ks + 64 + i * 32 + (g2 * 2 + q) * 8 + h * 4);
                            x[0] *= v4.x; x[1] *= v4.y; x[2] *= v4.z; x[3] *= v4.w;
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
        if (more) stage(mine + (cur ^ 1) * BUF, tile + KS);
        __syncthreads();
    }
    l += __shfl_xor(l, 32, 64);
    if constexpr (KS == 2) {
        // the second half's sums go to the first through LDS (nobody reads tiles any more), register by register
        float* x = reinterpret_cast<float*>(smem) + w4 * (16 * NT + 2) * 64 + lane;
        if (half) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[(j * 16 + e) * 64] = o[j][e];
            x[16 * NT * 64] = m;
            x[(16 * NT + 1) * 64] = l;
        }
        __syncthreads();
        if (half) return;
        const float m1 = x[16 * NT * 64], mn = fmaxf(m, m1), ms = mn == -INFINITY ? 0.f : mn;
        const float f0 = exp2_hw((m - ms) * unit), f1 = exp2_hw((m1 - ms) * unit);
        m = mn;
        l = l * f0 + x[(16 * NT + 1) * 64] * f1;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[j][e] = o[j][e] * f0 + x[(j * 16 + e) * 64] * f1;
    }
    if (wr0 + r32 >= rows) return;
    if (track && odd.any()) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[j][e] += odd.add(NT * (e / 4 * 8 + h * 4 + e % 4) + j, L);
    }
    const float mnat = BIAS ? m : m * a.scale;
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

// Joins the splits of a row: lane j has the maximum and sum of split j (there are at most 64), its weight goes to all lanes by v_readlane, and
// every split's output is requested without waiting for the one before.  WPR waves share the splits of a row (4 where there are many: a few
// rows of a long context would otherwise be one chain of 64 loads), and meet in LDS in their order.
template <int DK, int WPR>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttnArgs a) {
    constexpr int VEC = DK / 64;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = w % WPR;
    const int per = a.s.max_q * a.g;                                               // rows of a pair that may exist
    const long long row_id = (long long)blockIdx.x * (4 / WPR) + w / WPR;
    const int pair = (int)(row_id / per), rr = (int)(row_id % per);
    const int hk = pair % a.Hkv, b = pair / a.Hkv;
    if (b >= a.s.B) return;                                                        // (WPR = 4: the whole workgroup)
    const PagedSeq sq = paged_seq(a.s, b);
    if (rr >= min(sq.nq, a.s.max_q) * a.g) return;
    const size_t row = (size_t)(sq.q0 + rr / a.g) * a.H + hk * a.g + rr % a.g, step = (size_t)a.s.n_tok * a.H;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < a.splits) ml = *reinterpret_cast<const float2*>(a.part_ml + (lane * step + row) * 2);
    const int s0 = a.splits * part / WPR, s1 = a.splits * (part + 1) / WPR;
    constexpr int MOST = WPR == 4 ? 16 : 8;                                        // splits of a wave
    float x[MOST][VEC], acc[VEC] = {};
#pragma unroll
    for (int j = 0; j < MOST; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[j][i] = a.part_o[(min(s0 + j, a.splits - 1) * step + row) * DK + lane * VEC + i];
#pragma unroll
    for (int j = 0; j < MOST; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) arrived(x[j][i]);                            // (else each is requested where it is used)
    const float mx = wave_max(ml.x), ms = mx == -INFINITY ? 0.f : mx;
    const float f = exp2_hw((ml.x - ms) * LOG2E);
    const float sum = wave_sum(ml.y * f);
#pragma unroll
    for (int j = 0; j < MOST; ++j) {
        if (s0 + j >= s1) break;
        const float fs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s0 + j));
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = fmaf(x[j][i], fs, acc[i]);
    }
    if constexpr (WPR > 1) {
        __shared__ float so[WPR][DK];
#pragma unroll
        for (int i = 0; i < VEC; ++i) so[part][lane * VEC + i] = acc[i];
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int q = 1; q < WPR; ++q)
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] += so[q][lane * VEC + i];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    bf16_t* dst = a.out + (row / a.H) * a.o_st + (row % a.H) * DK + lane * VEC;
    if constexpr (VEC == 2) *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    else *dst = f32_to_bf16(acc[0] * inv);
    if (a.lse && lane == 0) a.lse[row] = sum == 0.f ? -INFINITY : mx + logf(sum);
}

template <int T, int DK, bool ODD>
void rows_launch(const PagedAttnArgs& a, unsigned blocks, int waves, int tiles, hipStream_t st) {
    if (waves == 1) hipLaunchKernelGGL((paged_attn_kernel<T, DK, 1, 1, ODD>), dim3(blocks), dim3(64), 0, st, a);
    else if (tiles == 1) hipLaunchKernelGGL((paged_attn_kernel<T, DK, 4, 1, ODD>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_attn_kernel<T, DK, 4, 2, ODD>), dim3(blocks), dim3(256), 0, st, a);
}
template <int T, int DK>
void rows_launch(const PagedAttnArgs& a, unsigned blocks, int waves, int tiles, hipStream_t st) {
    if (T != VLT5_KV_INT8 && a.causal && a.s.max_q > 1) rows_launch<T, DK, T != VLT5_KV_INT8>(a, blocks, waves, tiles, st);
    else rows_launch<T, DK, false>(a, blocks, waves, tiles, st);
}
template <int T, int DK, bool BIAS, int KS>
int chunk_launch(const PagedAttnArgs& a, unsigned blocks, hipStream_t st) {
    static std::atomic<unsigned long long> done{0};
    constexpr int bytes = 2 * KS * (64 * (DK * 2 + 16) + 4 * (DK / 32) * 1024 + 512) + (BIAS ? CHUNK_BIAS_LDS * 4 : 0) + (T == VLT5_KV_INT8 ? 0 : 8 * DK + 16);
    const int rc = vlt5_lds_optin((const void*)paged_chunk_kernel<T, DK, BIAS, KS>, bytes, done);
    if (rc) return rc;
    hipLaunchKernelGGL((paged_chunk_kernel<T, DK, BIAS, KS>), dim3(blocks), dim3(256 * KS), bytes, st, a);
    return VLT5_OK;
}

// query heads a multiple of the kv heads; rows are counted in 32 bits
bool paged_heads_ok(const vlt5_paged_attn_desc* d) {
    return d->H > 0 && d->H <= 1024 && d->H % d->kv.n_kv_heads == 0 && (long long)d->seqs.n_tok * d->H <= 0x7fffffffLL - 4096;
}
// The plan of a call, from what the host knows.
//   Up to 64 rows (tokens x heads of a group) go through the first kernel, more share their keys through LDS.  Where tiles of 16 rows fill the chip
//   (512 workgroups), 17 and more rows are better off reading every key once for two tiles (20 x 20 rows over 2000 keys 25.1 -> 20.1 us, 32 x 24 over
//   8000 152 -> 124, 41 x 40 over 10130 198 -> 182; a chip that is not full loses: 20 x 33 over 600 9.9 -> 12.3), in a bf16 cache, which has nothing
//   to convert, from 33 on through LDS (4 x 40 over 20000 81 -> 71, 100 x 33 over 400 36 -> 27; int8 182 -> 308).
//   A row tile's keys are shared by one wave up to 128 of them, else by four (80 x 58 keys, 12 heads: 6.0 against 8.0 us; 100 x 500: 20.4 against
//   19.1), and by as many workgroups as give every CU two, none with less than 512 keys (1 x 131071 keys, 8 kv heads of 128, int8: 63 us in 64
//   shares; 8 x 2000 keys: 15 us in 3 shares of 667, 17 in 7 of 286).
//   Large tiles that leave a CU one workgroup get twice the waves, half the keys each (8 x 200 tokens over 712 keys, 12 heads: 28.4 -> 20.5 us; where
//   CUs have two anyway it costs 5 %), and are shared out until every CU has that one (1 x 500 over 4000 33.6 -> 29.6; two a CU: twice the sums to
//   join), none with less than 341 keys (1 x 40 over 2000, 32 query and 4 kv heads of 128: 24.1 us with 512 and more, 20.2 with 341, 18.7 with 256;
//   2 x 128 over 3000, 8 heads: 25.0, 21.8, 25.9).
struct PagedPlan { int chunk, row_tiles, splits, waves, tiles; };              // tiles: of 16 rows that a wave of the first kernel takes
PagedPlan paged_plan(const vlt5_paged_attn_desc* d, const PagedSeqs& s) {
    const int g = d->H / d->kv.n_kv_heads;
    const long long rows = (long long)s.max_q * g, pairs = (long long)s.B * d->kv.n_kv_heads;
    const long long width = (long long)d->seqs.max_pages * d->kv.page_size, most_kv = d->max_kv > 0 && d->max_kv < width ? d->max_kv : width;
    auto share = [&](long long n, int parts) {                                 // ... of the keys between n workgroups, at least 1024 / parts for one
        const long long most = most_kv < VLT5_PAGED_SHARED_KV ? 1 : most_kv / (VLT5_PAGED_SHARED_KV / parts);
        n = n < most ? n : most;
        return (int)(n < 1 ? 1 : (n > 64 ? 64 : n));
    };
    PagedPlan p;
    auto small = [&](int tiles) {
        const long long n = (rows + 16 * tiles - 1) / (16 * tiles) * pairs;
        p.chunk = 0; p.tiles = tiles; p.row_tiles = (int)(n / pairs); p.splits = share((512 + n - 1) / n, 2); p.waves = most_kv <= 128 ? 1 : 4;
        return n * p.splits;
    };
    if (rows <= 64) {
        const bool full = small(1) >= 512;
        if (rows <= 16 || p.waves == 1 || !full) return p;
        if (rows <= 32 || d->kv.type != VLT5_KV_BF16) { small(2); return p; }
    }
    const long long n = (rows + 127) / 128 * pairs;
    p.chunk = 1; p.tiles = 0; p.row_tiles = (int)(n / pairs); p.splits = share(256 / n, 3); p.waves = n * p.splits <= 256 ? 8 : 4;
    return p;
}

}  // namespace

extern "C" long long vlt5_paged_attn_workspace_bytes(const vlt5_paged_attn_desc* d) {
    if (!d || vlt5_paged_check(&d->kv, &d->seqs) || !paged_heads_ok(d)) return -1;
    const PagedSeqs s = vlt5_paged_seqs_of(&d->kv, &d->seqs);
    const int sp = paged_plan(d, s).splits;
    return sp == 1 ? 0 : (long long)sp * s.n_tok * d->H * (d->kv.d_kv + 2) * 4;
}

extern "C" int vlt5_paged_attn(const vlt5_paged_attn_desc* d, void* stream) {
    if (!d || !d->q || !d->out) return VLT5_ERR_ARG;
    const int rc = vlt5_paged_check(&d->kv, &d->seqs);
    if (rc) return rc;
    const vlt5_paged_kv& c = d->kv;
    if (!paged_heads_ok(d)) return VLT5_ERR_ARG;
    if (d->q_st < (long long)d->H * c.d_kv || d->o_st < (long long)d->H * c.d_kv) return VLT5_ERR_ARG;
    if (d->rel_bias && (d->n_dist <= 0 || !d->causal || (long long)d->H * d->n_dist > 0x7fffffffLL)) return VLT5_ERR_ARG;      // (indexed in 32 bits)
    if (!(d->scale > 0.f && d->scale <= 3.402823466e38f)) return VLT5_ERR_ARG;
    if ((d->q_st & 7) || (d->o_st & 7) || (((uintptr_t)d->q | (uintptr_t)d->out | (uintptr_t)d->workspace) & 15)) return VLT5_ERR_ALIGN;
    // `out` may take q's place: a workgroup writes the very rows and heads that only it reads; over anything else others may still read it
    const RowSpan q = {d->q, d->seqs.n_tok, 2 * d->q_st, 2LL * d->H * c.d_kv}, out = {d->out, d->seqs.n_tok, 2 * d->o_st, q.width};
    const long long cache = (long long)c.n_kv_heads * c.page_size * c.d_kv * (c.type == VLT5_KV_BF16 ? 2 : 1);
    if (!(d->q == d->out && (d->q_st == d->o_st || d->seqs.n_tok == 1)) && vlt5_rows_overlap(out, q)) return VLT5_ERR_ARG;
    if (vlt5_rows_overlap(out, {c.k, c.n_pages, cache, cache}) || vlt5_rows_overlap(out, {c.v, c.n_pages, cache, cache})) return VLT5_ERR_ARG;
    if (d->seqs.n_tok == 0) return VLT5_OK;
    PagedAttnArgs a;
    a.s = vlt5_paged_seqs_of(&c, &d->seqs);
    a.k = (const unsigned char*)c.k; a.v = (const unsigned char*)c.v; a.ks = c.k_scale; a.vs = c.v_scale;
    a.q = (const bf16_t*)d->q; a.q_st = d->q_st; a.out = (bf16_t*)d->out; a.o_st = d->o_st; a.lse = d->lse;
    a.H = d->H; a.Hkv = c.n_kv_heads; a.g = d->H / c.n_kv_heads;
    a.scale = d->scale; a.causal = d->causal; a.bias = d->rel_bias; a.nd = d->n_dist;
    const PagedPlan plan = paged_plan(d, a.s);
    a.row_tiles = plan.row_tiles; a.splits = plan.splits;
    const long long rows = (long long)a.s.n_tok * a.H;
    if (a.splits > 1) {
        if (!d->workspace || d->workspace_bytes < (long long)a.splits * rows * (c.d_kv + 2) * 4) return VLT5_ERR_ARG;
        a.part_o = (float*)d->workspace;
        a.part_ml = a.part_o + (size_t)a.splits * rows * c.d_kv;
    } else {
        a.part_o = a.part_ml = nullptr;
    }
    const long long tiles = (long long)a.s.B * a.Hkv * a.row_tiles;
    const int wpr = a.splits > 8 ? 4 : 1;                                           // waves that join a row
    const long long joins = ((long long)a.s.B * a.H * a.s.max_q * wpr + 3) / 4;
    if (tiles * a.splits * (64 * plan.waves) > VLT5_MOST_THREADS || joins * 256 > VLT5_MOST_THREADS) return VLT5_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    int lrc = VLT5_OK;
#define PA(T, D) do { if (plan.chunk && plan.waves == 8) lrc = a.bias ? chunk_launch<T, D, true, 2>(a, (unsigned)(tiles * a.splits), st) : chunk_launch<T, D, false, 2>(a, (unsigned)(tiles * a.splits), st); \
                      else if (plan.chunk) lrc = a.bias ? chunk_launch<T, D, true, 1>(a, (unsigned)(tiles * a.splits), st) : chunk_launch<T, D, false, 1>(a, (unsigned)(tiles * a.splits), st); \
                      else rows_launch<T, D>(a, (unsigned)(tiles * a.splits), plan.waves, plan.tiles, st); } while (0)
    if (c.d_kv == 64) {
        if (c.type == VLT5_KV_BF16) PA(VLT5_KV_BF16, 64); else if (c.type == VLT5_KV_INT8) PA(VLT5_KV_INT8, 64); else PA(VLT5_KV_FP8, 64);
    } else {
        if (c.type == VLT5_KV_BF16) PA(VLT5_KV_BF16, 128); else if (c.type == VLT5_KV_INT8) PA(VLT5_KV_INT8, 128); else PA(VLT5_KV_FP8, 128);
    }
#undef PA
    if (lrc) return lrc;
    LAUNCH_CHECK();
    if (a.splits > 1) {
#define PJ(D, W) hipLaunchKernelGGL((paged_join_kernel<D, W>), dim3((unsigned)joins), dim3(256), 0, st, a)
        if (c.d_kv == 64) { if (wpr == 4) PJ(64, 4); else PJ(64, 1); }
        else { if (wpr == 4) PJ(128, 4); else PJ(128, 1); }
#undef PJ
        LAUNCH_CHECK();
    }
    return VLT5_OK;
}
