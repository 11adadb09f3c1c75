// Products of a few rows with 4-bit weights (the projections of a token-step, weight-only quantised).
//
//   out[m, n] = act(alpha * sum_k x[m, k] * value(code[n, k]) * scale[n, k / group] (+ resid[m, n]))
//
// Format of a weight [N, K]: byte j of row n holds k = 2j in its low four bits and k = 2j + 1 in the high ones; a code is an e2m1 number
// (sign, two exponent bits, one mantissa bit: 0 0.5 1 1.5 2 3 4 6), one bf16 scale per `group` consecutive k.  e2m1 and not a 4-bit integer:
// on normally distributed weights with the group's largest magnitude as the range both have the same rms error (0.11 sigma at 128), and
// gfx950 turns a pair of e2m1 codes into a pair of bf16 numbers in ONE instruction (v_cvt_scalef32_pk_bf16_fp4), exactly and with the sign,
// so the matrix instruction gets its operand with half an instruction per weight and no zero-point term has to be subtracted from the sums.
#include "common.h"
#include "rows.h"
#include "vlt5_hip.h"

namespace {

__device__ __forceinline__ uint32_t fp4_pair(uint32_t codes, int byte) {
    bf16_native2_t v;
    switch (byte) {
        case 0: v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 0); break;
        case 1: v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 1); break;
        case 2: v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 2); break;
        default: v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, 3); break;
    }
    return __builtin_bit_cast(uint32_t, v);
}
// eight codes (one dword) -> one MFMA operand
__device__ __forceinline__ bf16x8_t fp4x8(uint32_t codes) {
    const uint4 u = make_uint4(fp4_pair(codes, 0), fp4_pair(codes, 1), fp4_pair(codes, 2), fp4_pair(codes, 3));
    return __builtin_bit_cast(bf16x8_t, u);
}

// ---- quantiser -------------------------------------------------------------------------------------------------------------------
// One thread per eight consecutive k (a dword of codes), G / 8 neighbouring lanes per group.  scale = bf16(largest magnitude / 6), code =
// the nearest e2m1 number to w / scale in f32, ties to the even code.  A group that holds an infinity or a NaN gets the scale NaN: what it
// is multiplied with shows it.  A weight is quantised once, so this is plain code: eight scalar loads a lane, 32200 x 768 from f32 in 52 us (2.2 TB/s),
// 14336 x 4096 from bf16 in 108 us (1.4 TB/s).
template <int G>
__global__ __launch_bounds__(256) void quant_w4_kernel(const float* wf, const bf16_t* wb, long long ldw, int N, int K, int groups, uint32_t* codes,
                                                       bf16_t* scales) {
    const long long per_row = (long long)groups * (G / 8);
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const bool on = i < (long long)N * per_row;
    const int n = on ? (int)(i / per_row) : 0, k8 = on ? (int)(i % per_row) : 0;
    float v[8];
    float top = 0.f;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int k = k8 * 8 + e;
        v[e] = 0.f;
        if (on && k < K) v[e] = wf ? wf[(size_t)n * ldw + k] : bf16_to_f32(wb[(size_t)n * ldw + k]);
        bad |= !(fabsf(v[e]) <= 3.402823466e38f);
        top = fmaxf(top, fabsf(v[e]));
    }
#pragma unroll
    for (int o = 1; o < G / 8; o <<= 1) {
        top = fmaxf(top, __shfl_xor(top, o, 64));
        bad |= __shfl_xor((int)bad, o, 64) != 0;
    }
    const bf16_t sb = bad ? (bf16_t)0x7fc0 : f32_to_bf16(top / 6.0f);
    const float s = bf16_to_f32(sb);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float a = s > 0.f ? fabsf(v[e]) / s : 0.f;
        const uint32_t mag = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
        word |= (mag | (mag && v[e] < 0.f ? 8u : 0u)) << (4 * e);
    }
    if (on && k8 * 8 < K) codes[(size_t)n * (K / 8) + k8] = word;
    if (on && (k8 % (G / 8)) == 0) scales[(size_t)n * groups + k8 / (G / 8)] = sb;
}

// ---- product ---------------------------------------------------------------------------------------------------------------------
struct W4Args {
    const bf16_t* x; long long ldx;
    const unsigned char* codes; const bf16_t* scales;
    int rows, N, K, groups;
    float alpha;
    bf16_t* out_b; long long ldo;
    float* out_f; long long ldf;
    const float* resid; long long ldr;
    int relu;
    int splits; float* part;                   // > 1: the reduction in this many runs of chunks, their sums [splits][rows][N]
};

__device__ __forceinline__ void w4_store(const W4Args& a, int m, int n, float sum) {
    if (m >= a.rows || n >= a.N) return;
    float y = sum * a.alpha;
    if (a.resid) y += a.resid[(size_t)m * a.ldr + n];
    if (a.relu) y = y > 0.f ? y : (y != y ? y : 0.f);
    if (a.out_f) a.out_f[(size_t)m * a.ldf + n] = y;
    if (a.out_b) a.out_b[(size_t)m * a.ldo + n] = f32_to_bf16(y);
}

// A workgroup owns 16 rows and 8 / KW tiles of 16 columns; each tile's reduction is shared by KW waves in runs of neighbouring chunks of 128 k,
// whose sums meet in LDS in the order of the waves.  The rows of x are the A operand, the weights the B operand, so that a lane's four sums
// belong to ONE column and one scale serves them.  A reduction may be taken in any order as long as both operands agree, so the k that a lane
// holds follows the group length: the 32 k of one matrix instruction lie in one group, whose sum is scaled in f32 and added to the total.
//
// What bounds it at these sizes is not memory but the address unit: a load whose neighbouring lanes lie in different rows (the operand's own
// layout) costs 64 accesses instead of 16.  So nothing is loaded in operand layout: x goes to LDS once per workgroup in whole lines (row stride
// KS + 8 values: the sixteen rows of an operand start in sixteen bank groups), a chunk of codes (16 columns x 64 bytes) is loaded with four
// neighbouring lanes per column and turned round through one KB of LDS of the wave, and the scales of four chunks come with one load, one
// chunk per lane group.  Rows of x longer than LDS are taken in slabs of KS.  Against loads in operand layout (us per call in a replayed graph):
// 16 x 32200 x 768 11.1 -> 6.0, 1 x 4096 x 14336 11.0 -> 9.0 (29 MB: 5.4 TB/s less 3.3 us of launch), 200 x 5000 x 1024 22.2 -> 11.6; two or
// four row tiles per workgroup, sixteen waves, and a ring of more than four chunks were all slower.
template <int G, int KW>
__global__ __launch_bounds__(512) void w4_kernel(const W4Args a, int KS) {
    extern __shared__ __attribute__((aligned(16))) char w4_smem[];
    constexpr int GPC = 128 / G, DW = G / 32;                                  // groups per chunk, dwords of a lane per group
    constexpr int TW = 8 / KW, U = 4;                                          // column tiles; chunks requested ahead
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4;
    const int kw = w % KW;
    const int n_tile = (blockIdx.x * TW + w / KW) * 16, m_tile = blockIdx.y * 16;
    const int rows = min(16, a.rows - m_tile);
    char* turn = w4_smem + w * 1024;
    bf16_t* xs = reinterpret_cast<bf16_t*>(w4_smem + 8 * 1024);
    const int ld = KS + 8;
    // loads: lane l has piece (l & 3) of column l >> 2; LDS slot l, pieces swapped within the column so that the operand reads spread over the banks
    const int lcol = lane >> 2, lseg = (lane & 3) ^ ((lane >> 4) & 3);
    const unsigned char* wrow = a.codes + (size_t)min(n_tile + lcol, a.N - 1) * (a.K / 2);      // columns past the end repeat the last one, never stored
    const bf16_t* srow = a.scales + (size_t)min(n_tile + r16, a.N - 1) * a.groups;
    const bf16_t* xl = xs + min(r16, rows - 1) * ld;
    auto load_w = [&](int c) {                                                 // (a piece past the end of the row: any codes, x is zero there)
        return *reinterpret_cast<const vlt5_u32x4_t*>(wrow + c * 64 + (c * 128 + lseg * 32 < a.K ? lseg * 16 : 0));
    };
    struct Scales { bf16_t v[GPC]; };
    auto load_s = [&](int c, int end) {                                        // of chunk c + kq
        Scales s;
        const int at = min(c + kq, end - 1) * GPC;
        if (at + GPC <= a.groups) {
            __builtin_memcpy(&s, srow + at, sizeof s);
        } else {
#pragma unroll
            for (int i = 0; i < GPC; ++i) s.v[i] = srow[min(at + i, a.groups - 1)];
        }
        return s;
    };
    f32x4_t tot = {0.f, 0.f, 0.f, 0.f};
    const int all = (a.K + 127) / 128, start = (int)((long long)all * blockIdx.z / a.splits), chunks = (int)((long long)all * (blockIdx.z + 1) / a.splits);
    for (int cs = start; cs < chunks; cs += KS / 128) {
        const int cnt = min(KS / 128, chunks - cs);
        const int c0 = cs + cnt * kw / KW, c1 = cs + cnt * (kw + 1) / KW;
        vlt5_u32x4_t wr[U];
        Scales sn[U / 4];
        if (c0 < c1) {                                                         // on their way while x is staged
#pragma unroll
            for (int u = 0; u < U; ++u) if (c0 + u < c1) wr[u] = load_w(c0 + u);
#pragma unroll
            for (int q = 0; q < U / 4; ++q) sn[q] = load_s(c0 + q * 4, c1);
        }
        if (cs != start) __syncthreads();                                      // every wave is done with the slab before
        const int kmax = min(KS, a.K - cs * 128), pieces = (cnt * 128) / 8;
        for (int i0 = threadIdx.x; i0 < rows * pieces; i0 += 4 * 512) {
            uint4 v[4];
            int at[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int i = i0 + q * 512, r = i / pieces, k = (i - r * pieces) * 8;
                v[q] = make_uint4(0, 0, 0, 0);
                at[q] = i < rows * pieces ? r * ld + k : -1;
                if (at[q] >= 0 && k < kmax) v[q] = *reinterpret_cast<const uint4*>(a.x + (size_t)(m_tile + r) * a.ldx + cs * 128 + k);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (at[q] >= 0) *reinterpret_cast<uint4*>(xs + at[q]) = v[q];
        }
        __syncthreads();
        // one chunk: its codes through this wave's KB of LDS into the operand's layout (LDS operations of a wave complete in order: only the
        // compiler has to keep it), its scales from the lane group that has them
        auto multiply = [&](int c, const vlt5_u32x4_t& codes, const Scales& sc, int from) {
            __builtin_amdgcn_wave_barrier();
            *reinterpret_cast<vlt5_u32x4_t*>(turn + lane * 16) = codes;
            __builtin_amdgcn_wave_barrier();
            uint32_t sp[(GPC + 1) / 2];
            __builtin_memcpy(sp, &sc, sizeof sc);
#pragma unroll
            for (int i = 0; i < (GPC + 1) / 2; ++i) sp[i] = __builtin_amdgcn_ds_bpermute((from * 16 + r16) * 4, sp[i]);
#pragma unroll
            for (int gi = 0; gi < GPC; ++gi) {
                // this lane's codes of the group: 4 * DW bytes at gi * G / 2 + kq * 4 * DW of the column's 64
                const int byte = gi * (G / 2) + kq * (4 * DW);
                const char* p = turn + r16 * 64 + (((byte >> 4) ^ (r16 >> 2)) << 4) + (byte & 15);
                uint32_t cw[DW];
                __builtin_memcpy(cw, __builtin_assume_aligned(p, 4 * DW), sizeof cw);
                f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < DW; ++e) {
                    const bf16x8_t fx = *reinterpret_cast<const bf16x8_t*>(xl + (c - cs) * 128 + gi * G + kq * (8 * DW) + e * 8);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx, fp4x8(cw[e]), acc, 0, 0, 0);
                }
                const float s = __uint_as_float(gi & 1 ? sp[gi / 2] & 0xffff0000u : sp[gi / 2] << 16);
#pragma unroll
                for (int r = 0; r < 4; ++r) tot[r] = fmaf(s, acc[r], tot[r]);
            }
        };
        int c = c0;
        for (; c + 2 * U <= c1; c += U) {                                      // (every load unconditional, or the waits could not be counted)
            Scales sc[U / 4];
#pragma unroll
            for (int q = 0; q < U / 4; ++q) { sc[q] = sn[q]; sn[q] = load_s(c + U + q * 4, c1); }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                multiply(c + u, wr[u], sc[u / 4], u % 4);
                wr[u] = load_w(c + u + U);
            }
        }
        for (; c < c1; c += U) {
            Scales sc[U / 4];
#pragma unroll
            for (int q = 0; q < U / 4; ++q) { sc[q] = sn[q]; if (c + U < c1) sn[q] = load_s(c + U + q * 4, c1); }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (c + u >= c1) break;
                multiply(c + u, wr[u], sc[u / 4], u % 4);
                if (c + u + U < c1) wr[u] = load_w(c + u + U);
            }
        }
    }
    if constexpr (KW > 1) {
        __syncthreads();                                                       // codes and x are read no more: the sums take their place
        float4* red = reinterpret_cast<float4*>(w4_smem);
        red[w * 64 + lane] = make_float4(tot[0], tot[1], tot[2], tot[3]);
        __syncthreads();
        if (kw) return;
#pragma unroll
        for (int q = 1; q < KW; ++q) {
            const float4 o = red[(w + q) * 64 + lane];
            tot[0] += o.x; tot[1] += o.y; tot[2] += o.z; tot[3] += o.w;
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int m = m_tile + kq * 4 + r, n = n_tile + r16;
        if (a.splits == 1) w4_store(a, m, n, tot[r]);
        else if (m < a.rows && n < a.N) a.part[((size_t)blockIdx.z * a.rows + m) * a.N + n] = tot[r];
    }
}

// ---- product, many rows ----------------------------------------------------------------------------------------------------------
// Above 2^31 multiply-adds the kernel above is bound by its vector instructions: each code is converted and each sum scaled for sixteen rows, and long
// rows of x leave a CU one workgroup.  Here a workgroup has 32 rows and 128 columns, a wave 32 columns of them, on 32 x 32 x 16 instructions; chunks of
// 128 k of x go through two buffers of LDS (row stride 272 bytes: sixteen rows of an operand start in sixteen groups of four banks), the next two on
// their way while one is multiplied, codes and scales four chunks ahead, codes turned round through LDS as above.  The 16 k of an instruction lie in
// one group, half of them in each half of the wave.  256 x 4096 x 14336: 100 -> 58 us (0.52 PFLOP/s), 128 x 14336 x 4096 60 -> 31, 200 x 2000 x 8192
// 30 -> 23; what bounds it still is the vector unit (100 instructions a wave and chunk for 8 of the matrix unit).  64 rows a workgroup: 50, 33, 24.
typedef __attribute__((ext_vector_type(16))) float f32x16_t;

template <int G>
__global__ __launch_bounds__(256, 2) void w4_many_kernel(const W4Args a) {
    constexpr int GPC = 128 / G, DW = G / 16, KROW = 272, U = 4;               // groups of a chunk, dwords of a lane per group, chunks requested ahead
    __shared__ __attribute__((aligned(16))) char xs[2][32 * KROW];
    __shared__ __attribute__((aligned(16))) char turns[4][2048];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, r32 = lane & 31, h = lane >> 5;
    const int m_tile = blockIdx.y * 32, n0 = blockIdx.x * 128 + w * 32, n = n0 + r32;
    char* turn = turns[w];
    // loads as above: lane l has piece (l & 3), swapped within the column, of columns l >> 2 and 16 + (l >> 2); columns past the end repeat the last one
    const int lseg = (lane & 3) ^ ((lane >> 4) & 3);
    const unsigned char* wrow[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) wrow[j] = a.codes + (size_t)min(n0 + j * 16 + (lane >> 2), a.N - 1) * (a.K / 2);
    const bf16_t* srow = a.scales + (size_t)min(n, a.N - 1) * a.groups;
    const bf16_t* xrow[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) xrow[i] = a.x + (size_t)min(m_tile + i * 16 + (tid >> 4), a.rows - 1) * a.ldx;
    const int xk = (tid & 15) * 8;
    const int all = (a.K + 127) / 128, c0 = (int)((long long)all * blockIdx.z / a.splits), c1 = (int)((long long)all * (blockIdx.z + 1) / a.splits);
    uint4 xr[2][2];
    vlt5_u32x4_t cw[U][2];
    struct Scales { bf16_t v[2 * GPC]; } sn;
    // (past the end the last chunk again: every load unconditional, or the waits could not be counted; past the end of a row any codes, x is zero there)
    auto fetch_x = [&](int u, int c) {
        const int k = min(c, c1 - 1) * 128 + xk;
#pragma unroll
        for (int i = 0; i < 2; ++i) xr[u][i] = *reinterpret_cast<const uint4*>(xrow[i] + (k < a.K ? k : 0));
    };
    auto fetch_w = [&](int u, int past) {
        const int c = min(past, c1 - 1), at = c * 128 + lseg * 32 < a.K ? c * 64 + lseg * 16 : 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) cw[u][j] = *reinterpret_cast<const vlt5_u32x4_t*>(wrow[j] + at);
    };
    auto fetch_s = [&](int c) {                                                // of chunks c + 2 h and c + 2 h + 1
        const int at = (c + 2 * h) * GPC;
        if (at + 2 * GPC <= a.groups) {
            __builtin_memcpy(&sn, srow + at, sizeof sn);
        } else {
#pragma unroll
            for (int i = 0; i < 2 * GPC; ++i) sn.v[i] = srow[min(at + i, a.groups - 1)];
        }
    };
    auto stage = [&](int u, int c) {
        const bool past = c * 128 + xk >= a.K;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint4*>(xs[u] + (i * 16 + (tid >> 4)) * KROW + xk * 2) = past ? make_uint4(0, 0, 0, 0) : xr[u][i];
    };
    f32x16_t tot;
#pragma unroll
    for (int e = 0; e < 16; ++e) tot[e] = 0.f;
    fetch_x(0, c0);
    fetch_x(1, c0 + 1);
    fetch_s(c0);
#pragma unroll
    for (int u = 0; u < U; ++u) fetch_w(u, c0 + u);
    stage(0, c0);
    fetch_x(0, c0 + 2);
    __syncthreads();
    for (int c = c0; c < c1; c += U) {
        const Scales sc = sn;
        fetch_s(c + U);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (c + u >= c1) break;
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < 2; ++j) *reinterpret_cast<vlt5_u32x4_t*>(turn + j * 1024 + lane * 16) = cw[u][j];
            __builtin_amdgcn_wave_barrier();
            fetch_w(u, c + u + U);
            uint32_t sp[(GPC + 1) / 2];                                        // this chunk's scales, from the half that has them
            if constexpr (GPC == 1) {
                uint32_t both;
                __builtin_memcpy(&both, &sc, 4);
                both = __builtin_amdgcn_ds_bpermute(((u >> 1) * 32 + r32) * 4, both);
                sp[0] = u & 1 ? both >> 16 : both;
            } else {
                __builtin_memcpy(sp, &sc.v[(u & 1) * GPC], sizeof sp);
#pragma unroll
                for (int i = 0; i < GPC / 2; ++i) sp[i] = __builtin_amdgcn_ds_bpermute(((u >> 1) * 32 + r32) * 4, sp[i]);
            }
#pragma unroll
            for (int gi = 0; gi < GPC; ++gi) {
                uint32_t cg[DW];                                               // this lane's codes of the group: 4 * DW bytes at gi * G / 2 + h * G / 4 of the column's 64
#pragma unroll
                for (int q = 0; q < (DW + 3) / 4; ++q) {
                    const int byte = gi * (G / 2) + h * (G / 4) + q * 16;
                    const char* p = turn + r32 * 64 + (((byte >> 4) ^ ((r32 >> 2) & 3)) << 4) + (byte & 15);
                    constexpr int some = DW < 4 ? 4 * DW : 16;
                    __builtin_memcpy(cg + q * 4, __builtin_assume_aligned(p, some), some);
                }
                f32x16_t acc;
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
                for (int e = 0; e < DW; ++e)
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(xs[u & 1] + r32 * KROW + (gi * G + h * (G / 2) + e * 8) * 2), fp4x8(cg[e]), acc,
                                                                  0, 0, 0);
                const float s = __uint_as_float(gi & 1 ? sp[gi / 2] & 0xffff0000u : sp[gi / 2] << 16);
#pragma unroll
                for (int e = 0; e < 16; ++e) tot[e] = fmaf(s, acc[e], tot[e]);
            }
            if (c + u + 1 < c1) stage((u + 1) & 1, c + u + 1);
            fetch_x((u + 1) & 1, c + u + 3);
            __syncthreads();
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int m = m_tile + e / 4 * 8 + h * 4 + e % 4;
        if (a.splits == 1) w4_store(a, m, n, tot[e]);
        else if (m < a.rows && n < a.N) a.part[((size_t)blockIdx.z * a.rows + m) * a.N + n] = tot[e];
    }
}

// the runs of a split reduction, added in their order
__global__ __launch_bounds__(256) void w4_join_kernel(const W4Args a) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, all = (long long)a.rows * a.N;
    if (i >= all) return;
    float s = 0.f;
#pragma unroll 8
    for (int z = 0; z < a.splits; ++z) s += a.part[z * all + i];
    w4_store(a, (int)(i / a.N), (int)(i % a.N), s);
}

int w4_join(const W4Args& a, hipStream_t st) {
    if (a.splits > 1) {
        hipLaunchKernelGGL(w4_join_kernel, dim3((unsigned)(((long long)a.rows * a.N + 255) / 256)), dim3(256), 0, st, a);
        LAUNCH_CHECK();
    }
    return VLT5_OK;
}
template <int G, int KW>
int w4_launch(const W4Args& a, hipStream_t st) {
    static std::atomic<unsigned long long> done{0};
    const int rows = a.rows < 16 ? a.rows : 16;
    const int run = ((a.K + 127) / 128 + a.splits - 1) / a.splits * 128, room = 148 * 1024 / 2 / rows - 8;      // 8 KB of the 160 are for the codes on their way
    const int KS = run <= room ? run : room & ~127;
    const int rc = vlt5_lds_optin((const void*)w4_kernel<G, KW>, 160 * 1024, done);
    if (rc) return rc;
    const dim3 grid(((a.N + 15) / 16 + 8 / KW - 1) / (8 / KW), (a.rows + 15) / 16, a.splits);
    hipLaunchKernelGGL((w4_kernel<G, KW>), grid, dim3(512), 8 * 1024 + rows * (KS + 8) * 2, st, a, KS);
    LAUNCH_CHECK();
    return w4_join(a, st);
}
// How a reduction is shared.  Waves of a workgroup: as many as leave no more than one workgroup per CU (256), since what a workgroup stages is
// then read once per CU; never more than there are chunks.  Measured: 3 x 14336 x 4096 in 1 / 2 / 4 / 8 shares 15.7 / 11.6 / 11.3 / 13.9 us (rule:
// 2), 5 x 4097 x 14336 43.0 / 23.7 / 16.7 / 21.9 (4; with 8 the 257th workgroup runs alone), 80 x 2304 x 768 5.3 / 4.8 / 5.2 / 5.7 (2),
// 1 x 768 x 768 4.9 / 4.2 / 3.8 / 3.5 (8), 16 x 32200 x 768 6.0 / 7.1 / 9.3 / 13.3 (1).
// Workgroups: where a row tile of x is so long that reading it is what a workgroup spends its time on, the reduction is split for the price of a
// second launch: as many waves on columns as let 256 workgroups take runs of 96 KB and less, and no run much below 64 KB.
//   When: from 160 KB on (what does not fit LDS in one slab); VLT5_W4_SPLIT_BYTES where half the CUs idle; and where three in eight idle, from three
//   runs on if the tile and its workgroup's codes are 288 KB together.  Of some 550 sizes (1 - 64 rows, 500 - 8192 columns, 4096 - 16384 k), unsplit
//   against split, us, full chip: 6 x 4096 x 12288 (144 KB) 13.2 / 13.4, 6 x 4096 x 14336 (168) 15.5 / 14.7, 5 x 4096 x 16384 (160) 16.4 / 15.0;
//   half idle: 21 x 137 x 11552 17.4 / 8.8, 16 x 500 x 8192 12.4 / 8.1; 129 to 144 workgroups: 5 x 4097 x 14336 (364) 16.7 / 15.2, 5 x 4600 x 14336
//   16.5 / 15.5, 6 x 4368 x 12288 (336) 15.4 / 13.9, 64 x 4600 x 5088 (477) 22.6 / 18.1, 12 x 4097 x 6144 (240) 12.0 / 11.7, 8 x 4112 x 8192 (256, two
//   runs) 12.3 / 13.0, 4 x 4097 x 16384 (384, two runs) 17.0 / 17.9; 172 of them: 5 x 5500 x 14336 16.6 / 16.9.
//   How: two runs share a CU and take twice as long as one alone, so 256 workgroups are one round and the second 256 another; unsplit is as many
//   rounds as there are runs.  A workgroup for every run where that is fewer (two rounds where 256 workgroups have another way): 16 x 18000 x 8192
//   in 1 / 4 runs 32.7 / 27.3 (564 workgroups: three rounds for four), 16 x 23000 x 8192 37.2 / 33.5 (720), 16 x 25000 x 8192 38.6 / 38.3 (784: four),
//   16 x 21000 x 5120 in 1 / 3 runs 22.7 / 19.6 (495: two for three), 16 x 23000 x 5120 22.8 / 24.9 (540: three), 16 x 19000 x 12288 in 1 / 6 53.4 /
//   40.2 (894), 16 x 9400 x 14336 in 3 / 7 26.3 / 27.7 (222 against 518).
// More than 16 rows and 2^31 multiply-adds: the other kernel (kw 0), the reduction shared by up to 512 workgroups in runs of 1024 k and more; a chip with
// 192 workgroups shares only what is 8192 long (160 x 4096 x 4096 in 1 / 2 / 3 runs 23.3 / 22.3 / 21.6 us, 256 x 4096 x 14336 in 1 / 2 / 3 70 / 56 / 65,
// 64 x 14336 x 4096 in 1 / 2 24.9 / 28.2).  Below, it loses: 33 x 4096 x 4096 13.0 against 11.1, 256 x 2048 x 2304 14.4 / 10.4, 128 x 4096 x 4096 17.6 / 15.2.
struct W4Plan { int kw, splits; };
W4Plan w4_plan(int rows, int N, int K) {
    const long long tiles = (N + 15) / 16, blocks = (rows + 15) / 16;
    const int chunks = (K + 127) / 128;
    W4Plan p = {8, 1};
    if (rows > 16 && (double)rows * N * K > 2147483648.0) {
        const long long w = (N + 127LL) / 128 * ((rows + 31) / 32), most = 32LL * K < VLT5_W4_SPLIT_BYTES || (w >= 192 && chunks < 64) ? 1 : chunks / 8, share = 512 / w;
        p.kw = 0;
        p.splits = (int)(share < most ? share : most);
        if (p.splits < 1) p.splits = 1;
        return p;
    }
    while (p.kw > 1 && ((tiles * p.kw + 7) / 8 * blocks > 256 || p.kw / 2 >= chunks)) p.kw /= 2;
    auto wgs = [&](int kw) { return (tiles * kw + 7) / 8 * blocks; };
    auto rounds = [](long long n) { return n / 512 * 2 + (n % 512 + 255) / 256; };
    const long long bytes = 2LL * (rows < 16 ? rows : 16) * K, runs = (bytes + 65535) / 65536, codes = 64LL / p.kw * K;
    if (bytes >= 160 * 1024 || (wgs(p.kw) <= 128 && bytes >= VLT5_W4_SPLIT_BYTES) || (wgs(p.kw) <= 160 && runs >= 3 && bytes + codes >= 288 * 1024))
        for (int kw = p.kw; kw; kw /= 2) {
            const long long w = wgs(kw);
            long long sp = 256 / w;
            if (sp > runs || (kw == 1 && w <= 256 && bytes > sp * 96 * 1024 && (sp == 1 || w * runs <= 512) && rounds(w * runs) < runs)) sp = runs;
            if (sp > 1 && (kw == 1 || bytes <= sp * 96 * 1024)) {
                p.kw = kw; p.splits = (int)sp;
                break;
            }
        }
    return p;
}
template <int G>
int w4_shares(const W4Args& a, int kw, hipStream_t st) {
    if (kw == 0) {
        hipLaunchKernelGGL(w4_many_kernel<G>, dim3((a.N + 127) / 128, (a.rows + 31) / 32, a.splits), dim3(256), 0, st, a);
        LAUNCH_CHECK();
        return w4_join(a, st);
    }
    if (kw == 8) return w4_launch<G, 8>(a, st);
    if (kw == 4) return w4_launch<G, 4>(a, st);
    if (kw == 2) return w4_launch<G, 2>(a, st);
    return w4_launch<G, 1>(a, st);
}

}  // namespace

extern "C" int vlt5_quant_w4(const float* w_f32, const void* w_bf16, long long ldw, int N, int K, int group, void* codes, void* scales, void* stream) {
    if ((!w_f32) == (!w_bf16) || !codes || !scales || N <= 0 || K <= 0 || ldw < K) return VLT5_ERR_ARG;
    if (group != 32 && group != 64 && group != 128) return VLT5_ERR_ARG;
    if ((K & 31) || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 1)) return VLT5_ERR_ALIGN;
    const int groups = (K + group - 1) / group;
    const long long blocks = ((long long)N * groups * (group / 8) + 255) / 256;
    if (blocks * 256 > VLT5_MOST_THREADS) return VLT5_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
#define QW4(G) hipLaunchKernelGGL(quant_w4_kernel<G>, dim3((unsigned)blocks), dim3(256), 0, st, w_f32, (const bf16_t*)w_bf16, ldw, N, K, groups, (uint32_t*)codes, (bf16_t*)scales)
    if (group == 32) QW4(32);
    else if (group == 64) QW4(64);
    else QW4(128);
#undef QW4
    LAUNCH_CHECK();
    return VLT5_OK;
}

extern "C" long long vlt5_decode_linear_w4_workspace_bytes(int rows, int N, int K) {
    if (rows <= 0 || rows > VLT5_W4_MAX_ROWS || N <= 0 || N > 1 << 28 || K <= 0 || K > 1 << 28) return -1;
    const int sp = w4_plan(rows, N, K).splits;
    return sp == 1 ? 0 : 4LL * sp * rows * N;
}

extern "C" int vlt5_decode_linear_w4(const vlt5_decode_linear_w4_desc* d, void* stream) {
    if (!d || !d->x_bf16 || !d->codes || !d->scales || (!d->out_bf16 && !d->out_f32)) return VLT5_ERR_ARG;
    if (d->rows <= 0 || d->rows > VLT5_W4_MAX_ROWS || d->N <= 0 || d->N > 1 << 28 || d->K <= 0 || d->K > 1 << 28 || d->ldx < d->K) return VLT5_ERR_ARG;
    if (d->group != 32 && d->group != 64 && d->group != 128) return VLT5_ERR_ARG;
    if ((d->out_bf16 && d->ld_out_bf16 < d->N) || (d->out_f32 && d->ld_out_f32 < d->N) || (d->resid && d->ld_resid < d->N)) return VLT5_ERR_ARG;
    if ((d->K & 31) || (d->ldx & 7) || (((uintptr_t)d->x_bf16 | (uintptr_t)d->codes | (uintptr_t)d->workspace) & 15)) return VLT5_ERR_ALIGN;
    // what is written may not lie over what other workgroups still read; `resid` may be `out_f32`: its element is read by the lane that writes it
    const RowSpan x = {d->x_bf16, d->rows, 2 * d->ldx, 2LL * d->K}, ob = {d->out_bf16, d->rows, 2 * d->ld_out_bf16, 2LL * d->N};
    const RowSpan of = {d->out_f32, d->rows, 4 * d->ld_out_f32, 4LL * d->N}, res = {d->resid, d->rows, 4 * d->ld_resid, 4LL * d->N};
    const RowSpan codes = {d->codes, d->N, d->K / 2, d->K / 2}, scales = {d->scales, d->N, 2LL * ((d->K + d->group - 1) / d->group), 2LL * ((d->K + d->group - 1) / d->group)};
    const bool in_place = d->resid == d->out_f32 && (d->rows == 1 || d->ld_resid == d->ld_out_f32);
    if (vlt5_rows_overlap(ob, of) || (!in_place && vlt5_rows_overlap(of, res)) || vlt5_rows_overlap(ob, res)) return VLT5_ERR_ARG;
    for (const RowSpan& in : {x, codes, scales})
        if (vlt5_rows_overlap(ob, in) || vlt5_rows_overlap(of, in)) return VLT5_ERR_ARG;
    W4Args a;
    a.x = (const bf16_t*)d->x_bf16; a.ldx = d->ldx; a.codes = (const unsigned char*)d->codes; a.scales = (const bf16_t*)d->scales;
    a.rows = d->rows; a.N = d->N; a.K = d->K; a.groups = (d->K + d->group - 1) / d->group;
    a.alpha = d->alpha == 0.f ? 1.f : d->alpha;
    a.out_b = (bf16_t*)d->out_bf16; a.ldo = d->ld_out_bf16; a.out_f = d->out_f32; a.ldf = d->ld_out_f32;
    a.resid = d->resid; a.ldr = d->ld_resid; a.relu = d->relu;
    const W4Plan plan = w4_plan(a.rows, a.N, a.K);
    a.splits = plan.splits;
    a.part = (float*)d->workspace;
    if (plan.splits > 1 && (!d->workspace || d->workspace_bytes < vlt5_decode_linear_w4_workspace_bytes(a.rows, a.N, a.K))) return VLT5_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    if (d->group == 32) return w4_shares<32>(a, plan.kw, st);
    if (d->group == 64) return w4_shares<64>(a, plan.kw, st);
    return w4_shares<128>(a, plan.kw, st);
}
