"""CPU tests of the low-precision token-step's host side: descriptors mirror the header, the C entry points refuse what the kernels could
not take before anything is launched, and the wrappers refuse tensors that are not on the GPU."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from conftest import ROOT

ARG, ALIGN = 1001, 1002


@pytest.fixture(scope="module")
def built():
    import __graft_entry__ as ge
    ge.build()
    from vqacl_amd import _lib
    return _lib


def test_struct_sizes_match_the_c_side(built, tmp_path):
    names = {"vlt5_decode_linear_w4_desc": built.DecodeLinearW4Desc, "vlt5_paged_kv": built.PagedKV, "vlt5_paged_seqs": built.PagedSeqs,
             "vlt5_paged_attn_desc": built.PagedAttnDesc}
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "vlt5_hip.h"\nint main(void){' + "".join(f'printf("%zu\\n", sizeof({n}));' for n in names)
                   + 'printf("%zu %zu\\n", offsetof(vlt5_paged_attn_desc, scale), offsetof(vlt5_decode_linear_w4_desc, relu));return 0;}')
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = subprocess.check_output([str(exe)], text=True).split()
    assert [int(x) for x in got[:4]] == [C.sizeof(m) for m in names.values()]
    assert [int(x) for x in got[4:]] == [built.PagedAttnDesc.scale.offset, built.DecodeLinearW4Desc.relu.offset]


P = 4096            # a pointer that is never followed: every call below is refused on the host


def test_w4_refusals(built):
    f = built.lib().vlt5_decode_linear_w4
    ok = dict(x_bf16=P, ldx=64, codes=P, scales=P, rows=1, N=8, K=64, group=32, out_bf16=P, ld_out_bf16=8)
    assert f(None, None) == ARG
    for change, rc in (({"x_bf16": None}, ARG), ({"codes": None}, ARG), ({"scales": None}, ARG), ({"out_bf16": None}, ARG), ({"rows": 0}, ARG), ({"rows": 257}, ARG),
                       ({"N": 0}, ARG), ({"K": 0}, ARG), ({"group": 48}, ARG), ({"group": 256}, ARG), ({"ldx": 32}, ARG), ({"ld_out_bf16": 7}, ARG),
                       ({"out_f32": P, "ld_out_f32": 4}, ARG), ({"resid": P, "ld_resid": 4}, ARG), ({"K": 48, "ldx": 48}, ALIGN), ({"ldx": 68}, ALIGN),
                       ({"codes": P + 8}, ALIGN), ({"x_bf16": P + 2}, ALIGN)):
        d = built.DecodeLinearW4Desc(**{**ok, **change})
        assert f(C.byref(d), None) == rc, change
    # long rows for few columns: the reduction is split and needs a workspace of its own
    size = built.lib().vlt5_decode_linear_w4_workspace_bytes
    long = dict(ok, rows=16, K=8192, ldx=8192)
    need = size(16, 8, 8192)
    assert need > 0 and need % (4 * 16 * 8) == 0
    for change, rc in (({}, ARG), ({"workspace": P, "workspace_bytes": need - 1}, ARG), ({"workspace": P + 8, "workspace_bytes": need}, ALIGN)):
        assert f(C.byref(built.DecodeLinearW4Desc(**{**long, **change})), None) == rc, change
    edge = built.W4_SPLIT_BYTES
    assert f"#define VLT5_W4_SPLIT_BYTES {edge}\n" in open(os.path.join(ROOT, "include", "vlt5_hip.h")).read()
    assert size(16, 8, edge // 32 - 32) == 0 and size(16, 8, edge // 32) > 0 and size(1, 8, edge // 2) > 0 and size(16, 32200, 8192) == 0
    assert size(0, 8, 64) == size(257, 8, 64) == size(4, 0, 64) == size(4, 8, 0) == -1
    q = built.lib().vlt5_quant_w4
    assert q(None, None, 64, 4, 64, 32, P, P, None) == ARG and q(P, P, 64, 4, 64, 32, P, P, None) == ARG and q(P, None, 64, 4, 64, 33, P, P, None) == ARG
    assert q(P, None, 64, 0, 64, 32, P, P, None) == ARG and q(P, None, 32, 4, 64, 32, P, P, None) == ARG and q(P, None, 64, 4, 64, 32, None, P, None) == ARG
    assert q(P, None, 64, 4, 40, 32, P, P, None) == ALIGN and q(P, None, 64, 4, 64, 32, P + 4, P, None) == ALIGN


KV = dict(k=P, v=P, k_scale=P, v_scale=P, n_pages=4, n_kv_heads=2, d_kv=64, page_size=16, type=1)
SEQ = dict(table=P, kv_lens=P, cu_q=None, B=2, max_pages=3, n_tok=2, max_q=1)
BAD_KV = [({"k": None}, ARG), ({"v": None}, ARG), ({"k_scale": None}, ARG), ({"v_scale": None}, ARG), ({"n_pages": 0}, ARG), ({"n_kv_heads": 0}, ARG), ({"n_kv_heads": 2000}, ARG),
          ({"d_kv": 96}, ARG), ({"d_kv": 32}, ARG), ({"page_size": 8}, ARG), ({"page_size": 48}, ARG), ({"page_size": 2048}, ARG), ({"type": 3}, ARG), ({"type": -1}, ARG),
          ({"k": P + 8}, ALIGN), ({"v_scale": P + 4}, ALIGN)]
BAD_SEQ = [({"table": None}, ARG), ({"kv_lens": None}, ARG), ({"B": 0}, ARG), ({"B": 65536}, ARG), ({"max_pages": 0}, ARG), ({"n_tok": -1}, ARG), ({"n_tok": 3}, ARG), ({"max_q": -1}, ARG)]


def test_cache_refusals(built):
    L = built.lib()
    kv, seq = built.PagedKV(**KV), built.PagedSeqs(**SEQ)
    for change, rc in BAD_KV:
        bad = built.PagedKV(**{**KV, **change})
        assert L.vlt5_kv_page_write(C.byref(bad), C.byref(seq), P, 128, P, 128, None) == rc, change
        assert L.vlt5_kv_page_read(C.byref(bad), C.byref(seq), 4, P, P, None) == rc, change
    for change, rc in BAD_SEQ:
        bad = built.PagedSeqs(**{**SEQ, **change})
        assert L.vlt5_kv_page_write(C.byref(kv), C.byref(bad), P, 128, P, 128, None) == rc, change
        assert L.vlt5_kv_page_read(C.byref(kv), C.byref(bad), 4, P, P, None) == rc, change
    w, r = L.vlt5_kv_page_write, L.vlt5_kv_page_read
    a, s = C.byref(kv), C.byref(seq)
    assert w(None, s, P, 128, P, 128, None) == ARG and w(a, None, P, 128, P, 128, None) == ARG and w(a, s, None, 128, P, 128, None) == ARG
    assert w(a, s, P, 127, P, 128, None) == ARG and w(a, s, P, 132, P, 128, None) == ALIGN and w(a, s, P, 128, P + 2, 128, None) == ALIGN
    assert r(a, s, -1, P, P, None) == ARG and r(a, s, 4, None, P, None) == ARG and r(a, s, 4, P, P + 8, None) == ALIGN
    none = built.PagedSeqs(**{**SEQ, "n_tok": 0})
    assert w(a, C.byref(none), P, 128, P, 128, None) == 0 and r(a, s, 0, P, P, None) == 0                # nothing to do: nothing is launched


def test_attention_refusals(built):
    L = built.lib()
    ok = dict(q=P, q_st=256, out=P, o_st=256, H=4, scale=1.0, causal=1)

    def desc(kv={}, seq={}, **change):
        return built.PagedAttnDesc(kv=built.PagedKV(**{**KV, **kv}), seqs=built.PagedSeqs(**{**SEQ, **seq}), **{**ok, **change})
    assert L.vlt5_paged_attn(None, None) == ARG and L.vlt5_paged_attn_workspace_bytes(None) == -1
    for change, rc in BAD_KV:
        assert L.vlt5_paged_attn(C.byref(desc(kv=change)), None) == rc, change
        assert L.vlt5_paged_attn_workspace_bytes(C.byref(desc(kv=change))) == -1
    for change, rc in BAD_SEQ:
        assert L.vlt5_paged_attn(C.byref(desc(seq=change)), None) == rc, change
    for change, rc in (({"q": None}, ARG), ({"out": None}, ARG), ({"H": 3}, ARG), ({"H": 0}, ARG), ({"q_st": 255}, ARG), ({"o_st": 128}, ARG), ({"rel_bias": P}, ARG), ({"scale": 0.0}, ARG), ({"scale": -1.0}, ARG), ({"scale": float("nan")}, ARG), ({"scale": float("inf")}, ARG),
                       ({"rel_bias": P, "n_dist": 4, "causal": 0}, ARG), ({"q_st": 260}, ALIGN), ({"q": P + 2}, ALIGN), ({"out": P + 8}, ALIGN), ({"workspace": P + 4}, ALIGN)):
        assert L.vlt5_paged_attn(C.byref(desc(**change)), None) == rc, change
    # a long context of few sequences is shared out and needs a workspace of its own: too small is refused
    long = dict(seq={"max_pages": 4096})
    need = L.vlt5_paged_attn_workspace_bytes(C.byref(desc(**long)))
    assert need > 0 and need % (2 * 4 * (64 + 2) * 4) == 0
    assert L.vlt5_paged_attn(C.byref(desc(**long)), None) == ARG
    assert L.vlt5_paged_attn(C.byref(desc(**long, workspace=P, workspace_bytes=need - 1)), None) == ARG
    assert L.vlt5_paged_attn_workspace_bytes(C.byref(desc())) == 0
    edge = built.PAGED_SHARED_KV
    assert f"#define VLT5_PAGED_SHARED_KV {edge}\n" in open(os.path.join(ROOT, "include", "vlt5_hip.h")).read()
    assert L.vlt5_paged_attn_workspace_bytes(C.byref(desc(seq={"B": 1, "n_tok": 1, "max_pages": 4096}, max_kv=edge - 1))) == 0
    assert L.vlt5_paged_attn_workspace_bytes(C.byref(desc(seq={"B": 1, "n_tok": 1, "max_pages": 4096}, max_kv=edge))) > 0
    assert L.vlt5_paged_attn(C.byref(desc(seq={"n_tok": 0})), None) == 0


def test_a_bias_table_past_32_bits_is_refused(built):
    f = built.lib().vlt5_paged_attn
    for n_dist in (1 << 29, (1 << 29) + 1, 0x7fffffff):
        d = built.PagedAttnDesc(kv=built.PagedKV(**KV), seqs=built.PagedSeqs(**SEQ), q=P, q_st=256, out=P, o_st=256, H=4, scale=1.0, causal=1, rel_bias=P, n_dist=n_dist)
        assert f(C.byref(d), None) == ARG


def test_wrappers_refuse_host_tensors(built):
    from vqacl_amd import ops
    c = ops.KVPages(*(torch.zeros(2, 1, 16, 64, dtype=torch.int8) for _ in range(2)), *(torch.zeros(2, 1, 16) for _ in range(2)))
    t, n, x = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 64, dtype=torch.bfloat16)
    w = ops.W4Weight(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 1, dtype=torch.bfloat16), 64)
    for call in (lambda: ops.quant_w4(torch.zeros(4, 64)), lambda: ops.decode_linear_w4(x, w), lambda: ops.kv_page_write(c, x, x, t, n),
                 lambda: ops.kv_page_read(c, t, n, 4), lambda: ops.paged_attn(x, c, t, n)):
        with pytest.raises(built.Vlt5Error):
            call()


def test_the_plan_of_a_product_has_no_edge_beside_one_size(built):
    """A reduction is split by what a workgroup moves: neighbours in rows, columns and k are planned alike."""
    size = built.lib().vlt5_decode_linear_w4_workspace_bytes
    for N in range(4097, 5121, 31):
        for rows, K in ((5, 13504), (5, 14304), (5, 14336), (5, 15008), (6, 12288), (16, 7936), (14, 9600)):
            assert size(rows, N, K) > 0, (rows, N, K)
        for rows, K in ((4, 14336), (4, 16384), (3, 16384), (5, 10240), (8, 8192), (1, 14336)):
            assert size(rows, N, K) == 0, (rows, N, K)
    runs = lambda rows, N, K: size(rows, N, K) // (4 * rows * N)
    for N in range(16600, 24400, 200):                                                     # four runs for what unsplit takes as long as four: up to three rounds
        assert runs(16, N, 8192) == 4, N
    assert [runs(16, N, 5120) for N in (19000, 21000, 22000, 23000, 27000)] == [3, 3, 0, 0, 0]
    assert [runs(16, N, 14336) for N in (9000, 9400, 9900)] == [7, 3, 3]


def test_an_output_over_an_input_of_a_product_is_refused(built):
    """Other workgroups may still read what a workgroup would write; only `resid` may be the f32 output itself."""
    f = built.lib().vlt5_decode_linear_w4
    M, R, N, K = 1 << 30, 256, 8704, 1024                                                  # far apart: pointers that are never followed
    ok = dict(x_bf16=M, ldx=K, codes=2 * M, scales=3 * M, rows=R, N=N, K=K, group=32, out_bf16=4 * M, ld_out_bf16=N)
    wide = dict(ldx=K + N, ld_out_bf16=K + N)                                              # slices of one buffer
    f32 = dict(out_bf16=None, out_f32=4 * M, ld_out_f32=N)
    last = (R - 1) * 2
    for change in (dict(out_bf16=M), dict(out_bf16=M + 16), dict(out_bf16=M + last * K + 2 * K - 16), dict(out_bf16=M - last * N - 2 * N + 16), dict(wide, out_bf16=M + 2 * K - 16),
                   dict(wide, out_bf16=M - 2 * N + 16), dict(wide, out_bf16=M + last * (K + N) + 2 * K - 16), dict(out_bf16=M + 2 * N, ld_out_bf16=N + 8),
                   dict(out_bf16=2 * M + N * K // 2 - 16), dict(out_bf16=3 * M - last * N - 16), dict(out_f32=4 * M, ld_out_f32=N), dict(resid=4 * M, ld_resid=N),
                   dict(f32, out_f32=M), dict(f32, resid=4 * M + 4, ld_resid=N), dict(f32, resid=4 * M, ld_resid=N + 8)):
        d = built.DecodeLinearW4Desc(**{**ok, **change})
        assert f(C.byref(d), None) == ARG, change


def test_attention_over_its_own_queries_is_refused(built):
    """`out` may be `q`, row for row; a workgroup that writes elsewhere in q may be ahead of one that reads there."""
    f = built.lib().vlt5_paged_attn
    M = 1 << 20
    kv, seq = built.PagedKV(**{**KV, "k": 2 * M, "v": 3 * M}), built.PagedSeqs(**{**SEQ, "B": 3, "n_tok": 3})
    for change in (dict(out=M + 16), dict(out=M + 512), dict(out=M - 16), dict(out=M, o_st=264), dict(q_st=384, o_st=384, out=M + 128), dict(q_st=520, o_st=520, out=M - 16),
                   dict(out=M + 2 * 512 + 496), dict(out=2 * M + 4 * 2 * 16 * 64 - 16), dict(out=3 * M - 2 * 512 - 16)):
        d = built.PagedAttnDesc(**{**dict(kv=kv, seqs=seq, q=M, q_st=256, o_st=256, H=4, scale=1.0, causal=1), **change})
        assert f(C.byref(d), None) == ARG, change


def test_max_kv_past_the_table_counts_as_the_table(built):
    """No sequence can have more keys than its table: below VLT5_PAGED_SHARED_KV of them a call needs no workspace, whatever max_kv says."""
    size, most = built.lib().vlt5_paged_attn_workspace_bytes, built.PAGED_SHARED_KV

    def need(max_pages, max_kv, n_tok=1, H=4):
        return size(C.byref(built.PagedAttnDesc(kv=built.PagedKV(**KV), seqs=built.PagedSeqs(**{**SEQ, "B": 1, "n_tok": n_tok, "cu_q": P, "max_q": n_tok, "max_pages": max_pages}), q=P, q_st=256,
                                                out=P, o_st=256, H=H, scale=1.0, causal=1, max_kv=max_kv)))
    for n_tok in (1, 40, 700):
        for max_kv in (0, 1, most, 5000, 1 << 30):
            assert need(most // 16 - 1, max_kv, n_tok) == 0, (n_tok, max_kv)
            assert need(most // 16, max_kv, n_tok) == (0 if max_kv == 1 else need(most // 16, 0, n_tok)) and need(most // 16, 0, n_tok) > 0
            assert need(4096, max_kv, n_tok) >= need(most // 16, max_kv, n_tok)


def test_more_threads_than_a_grid_holds_are_refused(built):
    """A grid's threads are counted in 32 bits; without max_q it has room for every token in every sequence."""
    L = built.lib()
    kv = built.PagedKV(**{**KV, "n_kv_heads": 1024})
    many = built.PagedSeqs(**{**SEQ, "B": 65535, "n_tok": 65535, "max_pages": 16})
    d = dict(kv=kv, q=P, q_st=65536, out=1 << 44, o_st=65536, H=1024, scale=1.0, causal=1)
    assert L.vlt5_paged_attn(C.byref(built.PagedAttnDesc(seqs=many, **d)), None) == ARG
    kv = built.PagedKV(**{**KV, "n_kv_heads": 16, "d_kv": 128})
    long = built.PagedSeqs(**{**SEQ, "cu_q": P, "n_tok": 1 << 27, "max_q": 0})
    assert L.vlt5_kv_page_write(C.byref(kv), C.byref(long), P, 2048, P, 2048, None) == ARG
    assert L.vlt5_kv_page_read(C.byref(kv), C.byref(long), 1 << 27, P, P, None) == ARG
    assert L.vlt5_quant_w4(P, None, 1 << 20, 1 << 16, 1 << 20, 32, P, P, None) == ARG


def test_every_source_is_built_without_packed_f32_instructions():
    """Some forms of v_pk_add / mul / fma_f32 have given wrong results on this target now and then: the compiler is told to make none of them."""
    lines = subprocess.check_output(["make", "-C", os.path.join(ROOT, "vqacl_amd", "csrc"), "-n", "-B", "all", "exp"], text=True).splitlines()
    compiles = [line for line in lines if " -c " in line]
    sources = [f for f in os.listdir(os.path.join(ROOT, "vqacl_amd", "csrc")) if f.endswith(".hip")]
    assert len(compiles) == len(sources) + 1
    assert all("-Xclang -target-feature -Xclang -packed-fp32-ops" in line for line in compiles)
