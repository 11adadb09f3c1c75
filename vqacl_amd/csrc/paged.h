// Device side of the paged key/value cache: addresses, element types, operand conversions (csrc/paged.hip, csrc/paged_attn.hip).
#pragma once
#include "common.h"
#include "vlt5_hip.h"

// Where the rows of a sequence are.  Page ids, lengths and token offsets are DEVICE data that the host never sees: every one of them is
// held to its range here before an address is formed from it (a page id outside the cache = the page is not there, a length past the
// table = the table's length), so no content of these arrays can reach memory outside the tensors.
struct PagedSeqs {
    const int* table; int max_pages; int page_shift; int n_pages;
    const int* lens; const int* cu;
    int B, n_tok, max_q;
};

// csrc/paged.hip: host-side checks shared by the entry points of the cache, and the kernels' view of a call
int vlt5_paged_check(const vlt5_paged_kv* c, const vlt5_paged_seqs* q);
PagedSeqs vlt5_paged_seqs_of(const vlt5_paged_kv* c, const vlt5_paged_seqs* q);

struct PagedSeq {
    int q0, nq, len;          // first new token, number of new tokens, keys (new ones included)
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedSeqs& s, int b) {
    PagedSeq r;
    int q0 = s.cu ? s.cu[b] : b, q1 = s.cu ? s.cu[b + 1] : b + 1;
    q0 = min(max(q0, 0), s.n_tok);
    q1 = min(max(q1, q0), s.n_tok);
    r.q0 = q0; r.nq = q1 - q0;
    const long long most = min((long long)s.max_pages << s.page_shift, 0x7fff0000LL);
    r.len = (int)min((long long)max(s.lens[b], 0), most);
    return r;
}

// page of position `pos` of sequence b, or -1
__device__ __forceinline__ int paged_page(const PagedSeqs& s, int b, int pos) {
    const int p = s.table[(size_t)b * s.max_pages + (pos >> s.page_shift)];
    return (unsigned)p < (unsigned)s.n_pages ? p : -1;
}

// ---- element types ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cvt_fp8_pair(uint32_t w, bool hi) {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
}
__device__ __forceinline__ float sbyte(uint32_t w, int i) { return (float)(int)(signed char)(w >> (8 * i)); }

template <int T> struct KvType;                       // T: VLT5_KV_*
template <> struct KvType<VLT5_KV_BF16> { static constexpr int BYTES = 2; static constexpr bool SCALED = false; };
template <> struct KvType<VLT5_KV_INT8> { static constexpr int BYTES = 1; static constexpr bool SCALED = true; };
template <> struct KvType<VLT5_KV_FP8> { static constexpr int BYTES = 1; static constexpr bool SCALED = true; };

// four codes (one dword) -> two registers of bf16 pairs; every int8 and e4m3 value is exact in bf16
template <int T>
__device__ __forceinline__ uint2 codes_to_bf16(uint32_t w) {
    if constexpr (T == VLT5_KV_INT8) return make_uint2(pack_bf16x2(sbyte(w, 0), sbyte(w, 1)), pack_bf16x2(sbyte(w, 2), sbyte(w, 3)));
    else return make_uint2(cvt_fp8_pair(w, false), cvt_fp8_pair(w, true));
}
