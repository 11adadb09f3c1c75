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
// is multiplied with shows it.
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
};

// A workgroup owns 16 * NT columns and 16 * MT rows; its waves share the reduction in chunks of 128 k and meet in LDS.  The rows of x are the
// A operand, the weights the B operand, so that a lane's four sums belong to ONE column and one scale serves them.  A reduction may be
// taken in any order as long as both operands agree, so the k that a lane's dword stands for follows the group length: the 32 k of one
// matrix instruction must lie in one group, whose sum is scaled in f32 and added to the total.
template <int G, int MT, int NT>
__global__ __launch_bounds__(512) void w4_kernel(const W4Args a) {
    extern __shared__ __attribute__((aligned(16))) float4 w4_red[];            // [waves][MT][NT][64]
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, NW = blockDim.x >> 6;
    const int r16 = lane & 15, kq = lane >> 4;
    const int n_tile = blockIdx.x * (16 * NT), m_tile = blockIdx.y * (16 * MT);
    constexpr int GPC = 128 / G;                                               // groups per chunk
    constexpr int DW = 4 / GPC;                                                // dwords of a lane per group
    f32x4_t tot[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) tot[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int chunks = (a.K + 127) / 128;
    for (int c = w; c < chunks; c += NW) {
        uint32_t cw[NT][4];
        float sc[NT][GPC];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            int n = n_tile + j * 16 + r16;
            n = n < a.N ? n : a.N - 1;                                         // columns past the end repeat the last one, never stored
            const unsigned char* row = a.codes + (size_t)n * (a.K / 2);
#pragma unroll
            for (int gi = 0; gi < GPC; ++gi) {
                const int k = c * 128 + gi * G + kq * (8 * DW);
#pragma unroll
                for (int e = 0; e < DW; ++e) cw[j][gi * DW + e] = k + e * 8 < a.K ? *reinterpret_cast<const uint32_t*>(row + (k + e * 8) / 2) : 0u;
                sc[j][gi] = c * GPC + gi < a.groups ? bf16_to_f32(a.scales[(size_t)n * a.groups + c * GPC + gi]) : 0.f;
            }
        }
        f32x4_t acc[MT][NT];
#pragma unroll
        for (int gi = 0; gi < GPC; ++gi) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < DW; ++e) {
                const int k = c * 128 + gi * G + kq * (8 * DW) + e * 8;
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const int m = m_tile + i * 16 + r16;
                    bf16x8_t fx = {0, 0, 0, 0, 0, 0, 0, 0};
                    if (m < a.rows && k < a.K) fx = *reinterpret_cast<const bf16x8_t*>(a.x + (size_t)m * a.ldx + k);
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx, fp4x8(cw[j][gi * DW + e]), acc[i][j], 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) tot[i][j][r] = fmaf(sc[j][gi], acc[i][j][r], tot[i][j][r]);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) w4_red[((w * MT + i) * NT + j) * 64 + lane] = make_float4(tot[i][j][0], tot[i][j][1], tot[i][j][2], tot[i][j][3]);
    __syncthreads();
    for (int t = w; t < MT * NT; t += NW) {
        const int i = t / NT, j = t % NT;
        float4 v = w4_red[t * 64 + lane];
        for (int ww = 1; ww < NW; ++ww) {
            const float4 o = w4_red[(ww * MT * NT + t) * 64 + lane];
            v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
        }
        const int n = n_tile + j * 16 + r16;
        const float s[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int m = m_tile + i * 16 + kq * 4 + r;
            if (m >= a.rows || n >= a.N) continue;
            float y = s[r] * a.alpha;
            if (a.resid) y += a.resid[(size_t)m * a.ldr + n];
            if (a.relu) y = y > 0.f ? y : (y != y ? y : 0.f);
            if (a.out_f) a.out_f[(size_t)m * a.ldf + n] = y;
            if (a.out_b) a.out_b[(size_t)m * a.ldo + n] = f32_to_bf16(y);
        }
    }
}

template <int G, int MT, int NT>
int w4_launch(const W4Args& a, hipStream_t st) {
    const int chunks = (a.K + 127) / 128;
    const int NW = chunks >= 8 ? 8 : chunks;
    const dim3 grid((a.N + 16 * NT - 1) / (16 * NT), (a.rows + 16 * MT - 1) / (16 * MT));
    hipLaunchKernelGGL((w4_kernel<G, MT, NT>), grid, dim3(64 * NW), (size_t)NW * MT * NT * 1024, st, a);
    LAUNCH_CHECK();
    return VLT5_OK;
}
template <int G>
int w4_rows(const W4Args& a, hipStream_t st) {
    if (a.rows <= 16) return w4_launch<G, 1, 1>(a, st);
    if (a.rows <= 32) return w4_launch<G, 2, 1>(a, st);
    return w4_launch<G, 4, 1>(a, st);
}

}  // namespace

extern "C" int vlt5_quant_w4(const float* w_f32, const void* w_bf16, long long ldw, int N, int K, int group, void* codes, void* scales, void* stream) {
    if ((!w_f32) == (!w_bf16) || !codes || !scales || N <= 0 || K <= 0 || ldw < K) return VLT5_ERR_ARG;
    if (group != 32 && group != 64 && group != 128) return VLT5_ERR_ARG;
    if ((K & 31) || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 1)) return VLT5_ERR_ALIGN;
    const int groups = (K + group - 1) / group;
    const long long blocks = ((long long)N * groups * (group / 8) + 255) / 256;
    if (blocks > 0x7fffffffLL) return VLT5_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
#define QW4(G) hipLaunchKernelGGL(quant_w4_kernel<G>, dim3((unsigned)blocks), dim3(256), 0, st, w_f32, (const bf16_t*)w_bf16, ldw, N, K, groups, (uint32_t*)codes, (bf16_t*)scales)
    if (group == 32) QW4(32);
    else if (group == 64) QW4(64);
    else QW4(128);
#undef QW4
    LAUNCH_CHECK();
    return VLT5_OK;
}

extern "C" int vlt5_decode_linear_w4(const vlt5_decode_linear_w4_desc* d, void* stream) {
    if (!d || !d->x_bf16 || !d->codes || !d->scales || (!d->out_bf16 && !d->out_f32)) return VLT5_ERR_ARG;
    if (d->rows <= 0 || d->rows > VLT5_W4_MAX_ROWS || d->N <= 0 || d->K <= 0 || d->ldx < d->K) return VLT5_ERR_ARG;
    if (d->group != 32 && d->group != 64 && d->group != 128) return VLT5_ERR_ARG;
    if ((d->out_bf16 && d->ld_out_bf16 < d->N) || (d->out_f32 && d->ld_out_f32 < d->N) || (d->resid && d->ld_resid < d->N)) return VLT5_ERR_ARG;
    if ((d->K & 31) || (d->ldx & 7) || (((uintptr_t)d->x_bf16 | (uintptr_t)d->codes) & 15)) return VLT5_ERR_ALIGN;
    W4Args a;
    a.x = (const bf16_t*)d->x_bf16; a.ldx = d->ldx; a.codes = (const unsigned char*)d->codes; a.scales = (const bf16_t*)d->scales;
    a.rows = d->rows; a.N = d->N; a.K = d->K; a.groups = (d->K + d->group - 1) / d->group;
    a.alpha = d->alpha == 0.f ? 1.f : d->alpha;
    a.out_b = (bf16_t*)d->out_bf16; a.ldo = d->ld_out_bf16; a.out_f = d->out_f32; a.ldf = d->ld_out_f32;
    a.resid = d->resid; a.ldr = d->ld_resid; a.relu = d->relu;
    hipStream_t st = (hipStream_t)stream;
    if (d->group == 32) return w4_rows<32>(a, st);
    if (d->group == 64) return w4_rows<64>(a, st);
    return w4_rows<128>(a, st);
}
