"""GPU tests of the low-precision token-step: products with 4-bit weights (csrc/w4.hip), the paged key/value cache (csrc/paged.hip) and the
attention over it (csrc/paged_attn.hip), through vqacl_amd.ops, against plain 64-bit arithmetic on the same inputs.

Tolerances (u = 2^-24, half a step of f32; h = 2^-8, half a step of bf16, both relative to the value):
  product    a sum passes through at most G + groups + 16 f32 additions on its way (32 products and G / 32 instructions per group, the
             groups of a wave, the waves), each off by u of the magnitudes added so far: (G + groups + 16) u sum|x w|, then one rounding
  attention  a score s is a sum of d products: |ds| <= (d + 4) u scale sum|q k| + 2 u |s| + u (|s| + |bias|); the probability e^(s - m) is off by
             2 |ds| (score and maximum) + 2^-20 (the exponential and its argument), rounded once to bf16 (h); out adds one rounding (h |out|):
             |out - ref| <= (h + 4 max|ds| + 2^-18) sum p|v| + h |ref|
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F64 = torch.bfloat16, torch.float64
FP8 = torch.float8_e4m3fn
U, H = 2.0 ** -24, 2.0 ** -8
KINDS = [BF, torch.int8, FP8]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    from vqacl_amd import _lib
    _lib.lib()
    return torch.device("cuda", torch.cuda.current_device())


@pytest.fixture(scope="module")
def ops():
    from vqacl_amd import ops
    return ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- 4-bit weights --------------------------------------------------------------------------------------------------------------
E2M1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=F64)


def w4_value(w):
    """The weight that a W4Weight stands for, f64 on the CPU."""
    c = w.codes.cpu().long()
    n, k2 = c.shape
    v = torch.empty(n, 2 * k2, dtype=F64)
    v[:, 0::2], v[:, 1::2] = E2M1[c & 15], E2M1[c >> 4]
    return v * w.scales.cpu().double().repeat_interleave(w.group, 1)[:, :2 * k2]


@pytest.mark.parametrize("N,K,group,dtype", [(1, 32, 32, torch.float32), (17, 96, 64, BF), (33, 768, 128, torch.float32), (5, 160, 128, BF), (64, 4096, 32, BF)])
def test_quant_w4_takes_the_nearest_code(dev, ops, N, K, group, dtype):
    w = (torch.randn(N, K, generator=gen(N + K)) * torch.exp(torch.randn(N, 1, generator=gen(1)))).to(dtype)
    w[0, :7] = torch.tensor([6.0, 0.25, 0.75, -1.25, 1.75, -2.5, 5.0]).to(dtype)          # with the group's scale 1: ties
    w[0, 7:min(group, K)] = 0
    q = ops.quant_w4(w.to(dev), group)
    groups = -(-K // group)
    pad = torch.nn.functional.pad(w.float(), (0, groups * group - K)).view(N, groups, group)
    scale = (pad.abs().amax(-1) / 6.0).to(BF)
    assert torch.equal(q.scales.cpu(), scale)
    v = w4_value(q)
    s = scale.double().repeat_interleave(group, 1)[:, :K]
    ratio = torch.where(s > 0, w.double() / s, torch.zeros_like(s))
    best = (ratio.unsqueeze(-1) - E2M1).abs().amin(-1)                                  # distance to the nearest code, in units of the scale
    got = torch.where(s > 0, (ratio - v / torch.where(s > 0, s, 1.0)).abs(), torch.zeros_like(s))
    assert bool((got <= best + 8 * U * ratio.abs()).all())                               # (a quotient of f32 division may fall on the other side of a tie)
    assert (v[0, :7] == torch.tensor([6.0, 0.0, 1.0, -1.0, 2.0, -2.0, 4.0], dtype=F64)).all()


def test_quant_w4_shows_what_is_not_finite(dev, ops):
    w = torch.randn(4, 64, generator=gen(3))
    w[1, 5], w[2, 40], w[3] = float("nan"), float("inf"), 0
    q = ops.quant_w4(w.to(dev), 32)
    nan = torch.isnan(q.scales.cpu().float())
    assert nan.tolist() == [[False, False], [True, False], [False, True], [False, False]]
    y = ops.decode_linear_w4(torch.ones(1, 64, device=dev, dtype=BF), q).cpu()
    assert torch.isnan(y[0]).tolist() == [False, True, True, False] and float(y[0, 3]) == 0.0


@pytest.mark.parametrize("rows,N,K,group", [
    (1, 1, 32, 32), (1, 768, 768, 64), (2, 17, 96, 32), (5, 4097, 160, 128), (16, 100, 2048, 128), (17, 65, 800, 64), (31, 48, 32, 128),
    (33, 2304, 768, 128), (64, 7, 4128, 32), (65, 129, 1056, 64), (80, 768, 768, 32), (100, 33, 11008, 128), (129, 250, 320, 64), (256, 80, 544, 128),
])
@pytest.mark.parametrize("mode", ["bf16", "relu", "f32_resid"])
def test_decode_linear_w4(dev, ops, rows, N, K, group, mode):
    g = gen(rows * 7 + N + K)
    w = ops.quant_w4((torch.randn(N, K, generator=g) * K ** -0.5).to(dev), group)
    x = torch.randn(rows, K, generator=g).to(BF)
    v = w4_value(w)
    resid = torch.randn(rows, N, generator=g) if mode == "f32_resid" else None
    alpha = 0.5 if mode == "relu" else 1.0
    y = ops.decode_linear_w4(x.to(dev), w, alpha=alpha, relu=mode == "relu", resid=None if resid is None else resid.to(dev), out_f32=mode == "f32_resid").cpu().double()
    ref = alpha * x.double() @ v.t()
    acc = (group + -(-K // group) + 16) * U * alpha * (x.double().abs() @ v.abs().t())
    if resid is not None:
        ref = ref + resid.double()
        acc = acc + U * ref.abs()
    else:
        acc = acc + H * ref.abs()
    if mode == "relu":
        ref = ref.clamp_min(0)
    assert bool(((y - ref).abs() <= acc).all()), float(((y - ref).abs() / acc.clamp_min(1e-30)).max())


def test_decode_linear_w4_strides_and_in_place(dev, ops):
    g = gen(5)
    w = ops.quant_w4(torch.randn(70, 96, generator=g).to(dev), 32)
    wide = torch.randn(6, 3 * 96, generator=g).to(BF).to(dev)
    base = ops.decode_linear_w4(wide[:, 96:192].contiguous(), w)
    assert torch.equal(ops.decode_linear_w4(wide[:, 96:192], w), base)                    # a slice of a wider projection
    buf = torch.full((6, 80), 7.0, device=dev, dtype=BF)
    ops.decode_linear_w4(wide[:, 96:192], w, out=buf[:, 3:73])
    assert torch.equal(buf[:, 3:73], base) and bool((buf[:, :3] == 7).all()) and bool((buf[:, 73:] == 7).all())
    stream = torch.randn(6, 70, generator=g).to(dev)
    want = ops.decode_linear_w4(wide[:, 96:192], w, resid=stream, out_f32=True)
    got = stream.clone()
    assert ops.decode_linear_w4(wide[:, 96:192], w, resid=got, out=got) is got and torch.equal(got, want)      # the residual stream in place
    assert ops.decode_linear_w4(wide[:0, :96], w).shape == (0, 70)
    one = torch.zeros(1, 96, device=dev, dtype=BF)
    one[0, 3] = float("nan")
    assert bool(torch.isnan(ops.decode_linear_w4(one, w, relu=True)).all())
    assert torch.equal(ops.decode_linear_w4(wide[1:2, 96:192], w), base[1:2])             # a row's result does not depend on its neighbours


# ---- the cache ------------------------------------------------------------------------------------------------------------------
def make_cache(ops, dev, lens, heads, d, page, kind, seed, extra=2, fill=True):
    """A cache with shuffled pages, filled as earlier calls would have left it, and its block table (unused entries: -1)."""
    g = gen(seed)
    used = [-(-n // page) for n in lens]
    total = sum(used) + extra
    order = torch.randperm(total, generator=g)
    table = torch.full((len(lens), max(1, max(used))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at: at + n].to(torch.int32)
        at += n
    c = ops.kv_pages(total, heads, d, page, kind, dev)
    if fill:
        for pages, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
            x = torch.randn(total, heads, page, d, generator=g)
            codes, sc = plain_codes(x.to(BF), kind)
            raw(pages).copy_(raw(codes).to(dev))
            if scales is not None:
                scales.copy_(sc.to(dev))
    return c, table


def raw(t):
    return t.view(torch.uint8) if t.dtype == FP8 else t


def plain_codes(x, kind):
    """bf16 [..., d] -> codes and f32 scales by the cache's definition (f32 arithmetic, each operation rounded once)."""
    if kind == BF:
        return x, None
    most = 127.0 if kind == torch.int8 else 448.0
    x = x.float()
    sc = x.abs().amax(-1) / most
    y = torch.where(sc.unsqueeze(-1) > 0, x / sc.unsqueeze(-1), torch.zeros_like(x)).clamp(-most, most)
    return (torch.round(y).to(torch.int8) if kind == torch.int8 else y.to(FP8)), sc


def held(c, table, b, n):
    """Keys and values of sequence b by position, f64 on the CPU: two tensors [n, heads, d]; a page that is not there gives NaN."""
    page = c.k.shape[2]
    out = []
    for pages, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = pages.cpu().float().double()
        if scales is not None:
            x = x * scales.cpu().double().unsqueeze(-1)
        rows = [x[p, :, t % page] if 0 <= p < x.shape[0] else torch.full_like(x[0, :, 0], math.nan) for t in range(n) for p in [int(table[b, t // page])]]
        out.append(torch.stack(rows) if rows else x.new_zeros(0, x.shape[1], x.shape[3]))
    return out


def ints(dev, v):
    return torch.tensor(v, device=dev, dtype=torch.int32)


def starts(new):
    return [sum(new[:b]) for b in range(len(new) + 1)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,d,page,new,old", [
    (1, 64, 16, [1], [0]), (12, 64, 64, [58, 33, 0, 17], [0, 0, 0, 0]), (8, 128, 32, [5, 1, 40], [31, 32, 100]), (3, 128, 128, [130, 257], [1, 0]), (2, 64, 1024, [3], [1022]),
])
def test_kv_page_write_and_read(dev, ops, kind, heads, d, page, new, old):
    lens = [a + b for a, b in zip(new, old)]
    c, table = make_cache(ops, dev, lens, heads, d, page, kind, seed=heads + d)
    before = [None if t is None else raw(t).cpu().clone() for t in c]
    n = sum(new)
    both = torch.randn(n + 2, 2 * heads * d, generator=gen(n)) * torch.exp(torch.randn(n + 2, 1, generator=gen(9)))      # two rows of padding behind the last sequence
    both = both.to(BF)
    both[0, :d] = 0
    k, v = both[:, : heads * d], both[:, heads * d:]
    wide = both.to(dev)
    ops.kv_page_write(c, wide[:, : heads * d], wide[:, heads * d:], table.to(dev), ints(dev, lens), cu_q=ints(dev, starts(new)), max_q=max(new))
    want = [None if t is None else t.clone() for t in before]
    for x, pages, scales in ((k, 0, 2), (v, 1, 3)):
        codes, sc = plain_codes(x.reshape(n + 2, heads, d), kind)
        for b in range(len(new)):
            for i in range(new[b]):
                p, r = int(table[b, (old[b] + i) // page]), (old[b] + i) % page
                want[pages][p, :, r] = raw(codes)[starts(new)[b] + i]
                if sc is not None:
                    want[scales][p, :, r] = sc[starts(new)[b] + i]
    for got, exp in zip(c, want):
        assert (got is None and exp is None) or torch.equal(raw(got).cpu(), exp)             # every byte of the cache, rows of others included
    T = max(lens) + 3
    kr, vr = ops.kv_page_read(c, table.to(dev), ints(dev, lens), T)
    assert kr.shape == (len(new), T, heads * d)
    for b in range(len(new)):
        kk, vv = held(c, table, b, lens[b])
        for got, exp in ((kr, kk), (vr, vv)):
            got = got[b].cpu()
            assert torch.equal(got[: lens[b]].double(), exp.flatten(1).float().to(BF).double())       # code * scale rounded to f32, then to bf16
            assert bool((got[lens[b]:] == 0).all())
    if kind == torch.int8:                                                                  # half a step of the codes, then one bf16 rounding
        b, i = 0, new[0] - 1
        x = k[starts(new)[b] + i].double().view(heads, d)
        step = x.abs().amax(-1, keepdim=True) / 127
        back = kr[b, old[b] + i].cpu().double().view(heads, d)
        assert bool(((back - x).abs() <= 0.5 * step * (1 + 2.0 ** -18) + H * x.abs() + H * step).all())


@pytest.mark.parametrize("kind", [torch.int8, FP8])
def test_kv_rows_that_are_not_finite_or_tiny(dev, ops, kind):
    c = ops.kv_pages(1, 1, 64, 16, kind, dev)
    x = torch.randn(5, 64, generator=gen(2)).to(BF)
    x[0, 3], x[1, 63], x[2] = math.nan, -math.inf, 0
    x[3] = 1e-40                                                                            # subnormal: scale below the normal numbers
    x[4, 0] = 3.3e38
    t, n = ints(dev, [[0]]), ints(dev, [5])
    ops.kv_page_write(c, x.to(dev), x.to(dev), t, n, cu_q=ints(dev, [0, 5]))
    k, _ = ops.kv_page_read(c, t, n, 5)
    k = k[0].cpu().float()
    assert bool(torch.isnan(k[0]).all()) and bool(torch.isnan(k[1]).all()) and bool((k[2] == 0).all())
    codes, sc = plain_codes(x[3:], kind)
    assert torch.equal(k[3:], (codes.float() * sc.unsqueeze(-1)).to(BF).float())


def test_pages_that_are_not_there(dev, ops):
    """Bad page ids, lengths past the table and offsets past the tensors reach no memory: written nowhere, read as zeros, seen by nobody."""
    for kind in KINDS:
        c, _ = make_cache(ops, dev, [64], 2, 64, 16, kind, seed=1)
        before = [None if t is None else raw(t).clone() for t in c]
        n_pages = c.k.shape[0]
        x = torch.randn(3, 128, generator=gen(4)).to(BF).to(dev)
        for bad in (-1, n_pages, 2 ** 31 - 1, -2 ** 31):
            table = ints(dev, [[0, bad]])
            ops.kv_page_write(c, x, x, table, ints(dev, [20]), cu_q=ints(dev, [0, 3]))      # positions 17 .. 19: the missing page
            assert all(a is None or torch.equal(raw(a), b) for a, b in zip(c, before))
            k, _ = ops.kv_page_read(c, table, ints(dev, [20]), 20)
            assert bool((k[0, 16:] == 0).all()) and not bool((k[0, :16] == 0).all())
            full = ops.paged_attn(x[:1], c, table, ints(dev, [20]), causal=False)
            assert torch.equal(full, ops.paged_attn(x[:1], c, ints(dev, [[0, 1]]), ints(dev, [16]), causal=False))
        ops.kv_page_write(c, x, x, ints(dev, [[0]]), ints(dev, [40]), cu_q=ints(dev, [0, 3]))    # a length past the table counts as the table's: positions 13 .. 15
        k, _ = ops.kv_page_read(c, ints(dev, [[0]]), ints(dev, [99]), 18)
        assert not bool((k[0, 15] == 0).all()) and bool((k[0, 16:] == 0).all())
        for a, b in zip(c, before):
            if a is not None:
                raw(a).copy_(b)
        ops.kv_page_write(c, x, x, ints(dev, [[0]]), ints(dev, [-5]), cu_q=ints(dev, [0, 3]))    # no keys at all
        ops.kv_page_write(c, x, x, ints(dev, [[0], [1]]), ints(dev, [9, 9]), cu_q=ints(dev, [2 ** 31 - 1, -7, 3]), max_q=3)
        assert bool(torch.equal(raw(c.k)[0], before[0][0]))


# ---- attention over the cache -----------------------------------------------------------------------------------------------------
def attn_ref(q, c, table, new, lens, heads, scale, causal, bias):
    """(out, bound, lse) in f64, [tokens, heads, d] / [tokens, heads]."""
    hk, d = c.k.shape[1], c.k.shape[3]
    g = heads // hk
    n = sum(new)
    out, tol, lse = torch.zeros(n, heads, d, dtype=F64), torch.zeros(n, heads, d, dtype=F64), torch.full((n, heads), -math.inf, dtype=F64)
    for b in range(len(new)):
        k, v = held(c, table, b, lens[b])
        gone = torch.isnan(k).any(-1).any(-1)
        k, v = torch.nan_to_num(k), torch.nan_to_num(v)
        dist = torch.arange(lens[b] - new[b], lens[b])[:, None] - torch.arange(lens[b])[None]
        seen = ((dist >= 0) if causal else torch.ones_like(dist, dtype=torch.bool)) & ~gone
        for h in range(heads):
            rows = slice(starts(new)[b], starts(new)[b + 1])
            qh, kh, vh = q[rows].view(-1, heads, d)[:, h].double(), k[:, h // g], v[:, h // g]
            s = qh @ kh.t() * scale
            ds = (d + 4) * U * abs(scale) * (qh.abs() @ kh.abs().t()) + 2 * U * s.abs()
            if bias is not None:
                add = bias[h].double()[dist.clamp(0, bias.shape[1] - 1)]
                s = s + add
                ds = ds + U * (s.abs() + torch.nan_to_num(add.abs(), posinf=0.0))
            s = s.masked_fill(~seen, -math.inf)
            ds = torch.where(seen & (s > -1e30), ds, torch.zeros_like(ds))
            if s.numel() == 0:
                continue
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
            tot = p.sum(-1, keepdim=True)
            p = p / torch.where(tot > 0, tot, torch.ones_like(tot))
            out[rows, h] = p @ vh
            tol[rows, h] = (H + 4 * ds.amax(-1, keepdim=True) + 2.0 ** -18) * (p @ vh.abs()) + H * out[rows, h].abs()
            lse[rows, h] = (top + tot.log()).squeeze(-1)
    return out, tol, lse


def check_attn(ops, dev, c, table, new, lens, heads, *, scale=None, causal=True, bias=None, seed=0, max_kv=None, pad=3):
    d = c.k.shape[3]
    n = sum(new)
    scale = d ** -0.5 if scale is None else scale
    wide = torch.randn(n + pad, heads * d + 64, generator=gen(seed + n)).to(BF)
    q = wide[:, : heads * d]
    out = torch.full((n + pad, heads * d), 5.0, device=dev, dtype=BF)
    single = all(x == 1 for x in new)
    if single and seed % 2 == 0:
        pad = 0
        got, lse = ops.paged_attn(wide.to(dev)[:n, : heads * d], c, table.to(dev), ints(dev, lens), scale=scale, causal=causal, rel_bias=None if bias is None else bias.to(dev),
                                  max_kv=max_kv, out=out[:n], want_lse=True)
    else:
        got, lse = ops.paged_attn(wide.to(dev)[:, : heads * d], c, table.to(dev), ints(dev, lens), cu_q=ints(dev, starts(new)), max_q=max(new), scale=scale, causal=causal,
                                  rel_bias=None if bias is None else bias.to(dev), max_kv=max_kv, out=out, want_lse=True)
    assert bool((out[n:] == 5.0).all())                                                     # rows behind the last sequence keep what they held
    ref, tol, rl = attn_ref(q[:n], c, table, new, lens, heads, scale, causal, bias)
    err = (got[:n].cpu().double().view(n, heads, d) - ref).abs()
    assert bool(torch.isfinite(got[:n]).all())
    assert bool((err <= tol + 1e-30).all()), float((err / tol.clamp_min(1e-30)).max())
    lse = lse[:n].cpu().double()
    assert torch.equal(lse == -math.inf, rl == -math.inf)
    fin = rl > -math.inf
    assert bool(((lse - rl).abs()[fin] <= 1e-5 * (1 + rl.abs()[fin])).all())
    return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hk,g,page,lens", [
    (1, 1, 16, [1]), (2, 1, 16, [17, 1, 0, 64]), (2, 3, 64, [65, 128, 100]), (1, 16, 32, [333, 5]), (1, 20, 128, [257]), (4, 8, 64, [0]), (2, 4, 16, [3000, 700, 1]),
])
def test_single_tokens(dev, ops, kind, d, hk, g, page, lens):
    c, table = make_cache(ops, dev, lens, hk, d, page, kind, seed=sum(lens) + d)
    for causal in (True, False):
        check_attn(ops, dev, c, table, [1] * len(lens), lens, hk * g, causal=causal, seed=2 * g + (hk == 2))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hk,g,page,new,lens", [
    (2, 1, 16, [2, 0, 7], [2, 9, 100]), (1, 2, 64, [33, 1], [33, 300]), (2, 4, 32, [16, 65], [80, 65]), (1, 1, 64, [130], [513]), (1, 3, 128, [200, 77], [700, 90]), (2, 8, 16, [70], [71]),
])
def test_chunks(dev, ops, kind, d, hk, g, page, new, lens):
    c, table = make_cache(ops, dev, lens, hk, d, page, kind, seed=sum(lens) + d)
    for causal in (True, False):
        check_attn(ops, dev, c, table, new, lens, hk * g, causal=causal, seed=g)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,g,new,nd", [(64, 1, 20, 0), (64, 3, 13, 40), (64, 1, 63, 0), (128, 1, 17, 0), (128, 4, 10, 16), (128, 2, 32, 0)])
def test_few_rows_on_a_full_chip(dev, ops, kind, d, g, new, nd):
    """Enough sequences that two row tiles share the keys they read: 17 to 64 rows, ragged, with empty sequences and one whose keys end inside a step."""
    B, hk = 66, 8
    lens = [170 - (7 * b) % 90 for b in range(B)]
    news = [max(0, min(n, new - (b % 5) * (new // 6))) for b, n in enumerate(lens)]
    news[3] = lens[4] = news[4] = 0
    c, table = make_cache(ops, dev, lens, hk, d, 16, kind, seed=new + d)
    bias = 2 * torch.randn(hk * g, nd, generator=gen(nd)) if nd else None
    check_attn(ops, dev, c, table, news, lens, hk * g, scale=1.0 if nd else None, bias=bias, seed=1)


@pytest.mark.parametrize("new,lens,nd", [([1, 1, 1], [1, 40, 300], 32), ([1, 1], [2000, 129], 128), ([20, 150], [20, 400], 128), ([65], [1000], 1), ([3], [70], 500)])
@pytest.mark.parametrize("kind", KINDS)
def test_relative_bias(dev, ops, kind, new, lens, nd):
    c, table = make_cache(ops, dev, lens, 4, 64, 16, kind, seed=nd)
    check_attn(ops, dev, c, table, new, lens, 4, scale=1.0, bias=3 * torch.randn(4, nd, generator=gen(nd)), seed=1)


def test_bias_of_the_lowest_value_and_minus_infinity(dev, ops):
    lens, new = [40, 90], [5, 3]
    c, table = make_cache(ops, dev, lens, 2, 64, 16, torch.int8, seed=8)
    low = torch.finfo(torch.float32).min
    for nd, far in ((8, low), (8, -math.inf), (64, low)):                                    # keys further than nd - 1 count for nothing
        bias = torch.randn(2, nd, generator=gen(nd))
        bias[:, 6:] = far
        check_attn(ops, dev, c, table, new, lens, 2, bias=bias, seed=3)
    # all of a row at -inf: no key, zeros
    out, lse = ops.paged_attn(torch.randn(8, 128, generator=gen(1)).to(BF).to(dev), c, table.to(dev), ints(dev, lens), cu_q=ints(dev, [0, 5, 8]),
                              rel_bias=torch.full((2, 1), -math.inf, device=dev), want_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    # all of a row at the lowest value: the scores vanish in it and every visible key weighs the same
    out = ops.paged_attn(torch.randn(8, 128, generator=gen(1)).to(BF).to(dev), c, table.to(dev), ints(dev, lens), cu_q=ints(dev, [0, 5, 8]),
                         rel_bias=torch.full((2, 1), low, device=dev)).cpu().double().view(8, 2, 64)
    _, v = held(c, table, 1, 90)
    assert bool(((out[7] - v.mean(0)).abs() <= H * v.abs().mean(0) * 2 + H * v.mean(0).abs()).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1], [40, 9]])
def test_what_lies_behind_the_last_key_does_not_matter(dev, ops, kind, new):
    lens = [75, 9]
    c, table = make_cache(ops, dev, lens, 2, 64, 16, kind, seed=6)
    clean = check_attn(ops, dev, c, table, new, lens, 4, seed=1)
    for b in range(2):
        p, r = int(table[b, lens[b] // 16]), lens[b] % 16
        for pages, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
            if kind == torch.int8:
                pages[p, :, r:] = 127
            else:
                raw(pages)[p, :, r:] = math.nan if kind == BF else 0x7f
            if scales is not None:
                scales[p, :, r:] = math.nan if b else math.inf
    assert torch.equal(check_attn(ops, dev, c, table, new, lens, 4, seed=1), clean)


def test_holes_in_the_table(dev, ops):
    lens, new = [200, 130], [20, 1]
    for kind in KINDS:
        c, table = make_cache(ops, dev, lens, 2, 64, 16, kind, seed=12)
        table[0, 1], table[0, 5], table[1, 0:8] = -1, c.k.shape[0], -7
        check_attn(ops, dev, c, table, new, lens, 4, seed=1)
        check_attn(ops, dev, c, table, [1, 1], lens, 4, seed=1)
        table[1, 8] = -1
        out, lse = ops.paged_attn(torch.ones(2, 256, device=dev, dtype=BF), c, table.to(dev), ints(dev, lens), want_lse=True)
        assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all()) and bool(torch.isfinite(lse[0]).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 5, 70])
def test_the_split_changes_nothing_but_roundings(dev, ops, kind, new):
    """One sequence with a long context: its keys are shared out; the hint that decides how is no limit."""
    lens = [9001]
    c, table = make_cache(ops, dev, lens, 2, 128, 64, kind, seed=13)
    for max_kv in (None, 64, 9001):
        check_attn(ops, dev, c, table, [new], lens, 8, max_kv=max_kv, seed=1)


def test_a_long_cache_past_32_bit_offsets(dev, ops):
    """The last pages of a cache of more than 2^32 bytes a tensor."""
    pages, hk, d, page = 2 ** 18 + 8, 2, 128, 64
    c = ops.KVPages(*(torch.empty(pages, hk, page, d, device=dev, dtype=torch.int8) for _ in range(2)), *(torch.empty(pages, hk, page, device=dev) for _ in range(2)))
    assert c.k.numel() > 2 ** 32
    lens, new = [130, 70], [130, 70]
    table = torch.tensor([[pages - 1, 5, pages - 3], [pages - 2, 0, -1]], dtype=torch.int32)
    kv = torch.randn(200, 2 * hk * d, generator=gen(1)).to(BF).to(dev)
    ops.kv_page_write(c, kv[:, : hk * d], kv[:, hk * d:], table.to(dev), ints(dev, lens), cu_q=ints(dev, starts(new)))
    small = ops.KVPages(*(t[[pages - 1, 5, pages - 3, pages - 2, 0]].contiguous() for t in c))
    near = torch.tensor([[0, 1, 2], [3, 4, -1]], dtype=torch.int32)
    k, v = ops.kv_page_read(c, table.to(dev), ints(dev, lens), 130)
    ks, vs = ops.kv_page_read(small, near.to(dev), ints(dev, lens), 130)
    assert torch.equal(k, ks) and torch.equal(v, vs) and not bool((k[0] == 0).all(-1).any())
    q = torch.randn(200, 4 * d, generator=gen(2)).to(BF).to(dev)
    for kw in (dict(cu_q=ints(dev, starts(new))), {}):
        rows = q if kw else q[:2]
        assert torch.equal(ops.paged_attn(rows, c, table.to(dev), ints(dev, lens), scale=0.1, **kw), ops.paged_attn(rows, small, near.to(dev), ints(dev, lens), scale=0.1, **kw))


def test_two_streams_and_a_replayed_graph(dev, ops):
    """Calls in flight on two streams, and a captured step whose inputs change between the replays, give what the eager calls give."""
    lens = [4000, 2500]
    c, table = make_cache(ops, dev, lens, 2, 64, 16, torch.int8, seed=3)
    t, n = table.to(dev), ints(dev, lens)
    w = ops.quant_w4(torch.randn(512, 512, generator=gen(1)).to(dev), 64)
    kv = torch.randn(2, 256, generator=gen(2)).to(BF).to(dev)

    def step(x):
        q = ops.decode_linear_w4(x, w)
        ops.kv_page_write(c, kv[:, :128], kv[:, 128:], t, n)
        return ops.decode_linear_w4(ops.paged_attn(q, c, t, n), w, out_f32=True)
    xs = [torch.randn(2, 512, generator=gen(10 + i)).to(BF).to(dev) for i in range(6)]
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    lanes = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i, x in enumerate(xs):
        with torch.cuda.stream(lanes[i % 2]):
            got.append(step(x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(x)
    for i in (3, 1, 5, 0):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])
        assert torch.equal(step(xs[2]), want[2])                                            # eager work between the replays


# ---- together: the self-attention sublayer of a decoder, a prompt and then tokens one by one ------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
def test_a_decoder_sublayer_in_low_precision(dev, ops, kind):
    """q | k | v in four bits, keys and values into the pages, attention with T5's relative bias, the output product onto the residual stream:
    a ragged prompt chunk, then single tokens, each step against 64-bit arithmetic on what the step before left (the bf16 activations and
    the cache's codes), so that every operator is held to its own bound."""
    B, heads, d, dm, page = 3, 4, 64, 256, 16
    g = gen(21)
    wq = ops.quant_w4((torch.randn(3 * heads * d, dm, generator=g) * dm ** -0.5).to(dev), 64)
    wo = ops.quant_w4((torch.randn(dm, heads * d, generator=g) * (heads * d) ** -0.5).to(dev), 64)
    vq, vo = w4_value(wq), w4_value(wo)
    bias = torch.randn(heads, 32, generator=g)
    total = [37 + 4, 16 + 4, 1 + 4]
    c, table = make_cache(ops, dev, total, heads, d, page, kind, seed=22, fill=False)
    lens = [0, 0, 0]
    for new in ([37, 16, 1], [1, 1, 1], [1, 1, 1], [1, 1, 1], [1, 1, 1]):
        n = sum(new)
        lens = [a + b for a, b in zip(lens, new)]
        x = torch.randn(n, dm, generator=g)
        xb = x.to(BF)
        cu = None if n == 3 else ints(dev, starts(new))
        qkv = ops.decode_linear_w4(xb.to(dev), wq)
        ref = xb.double() @ vq.t()
        assert bool(((qkv.cpu().double() - ref).abs() <= (64 + 4 + 16) * U * (xb.double().abs() @ vq.abs().t()) + H * ref.abs()).all())
        inner = heads * d
        ops.kv_page_write(c, qkv[:, inner: 2 * inner], qkv[:, 2 * inner:], table.to(dev), ints(dev, lens), cu_q=cu)
        for b in range(B):
            kk, vv = held(c, table, b, lens[b])
            mine = slice(starts(new)[b], starts(new)[b + 1])
            for got, part in ((kk, qkv[mine, inner: 2 * inner]), (vv, qkv[mine, 2 * inner:])):
                codes, sc = plain_codes(part.cpu().view(-1, heads, d), kind)
                exp = codes.float().double() * (1.0 if sc is None else sc.double().unsqueeze(-1))
                assert torch.equal(got[lens[b] - new[b]:], exp)
        ctx = ops.paged_attn(qkv[:, :inner], c, table.to(dev), ints(dev, lens), cu_q=cu, rel_bias=bias.to(dev))
        ref, tol, _ = attn_ref(qkv[:, :inner].cpu(), c, table, new, lens, heads, 1.0, True, bias)
        assert bool(((ctx.cpu().double().view(n, heads, d) - ref).abs() <= tol).all())
        stream = x.to(dev)
        ops.decode_linear_w4(ctx, wo, resid=stream, out=stream)
        cb = ctx.cpu().double()
        ref = cb @ vo.t() + x.double()
        assert bool(((stream.cpu().double() - ref).abs() <= (64 + 4 + 16) * U * (cb.abs() @ vo.abs().t()) + U * ref.abs()).all())


# ---- refusals -------------------------------------------------------------------------------------------------------------------
def test_refusals(dev, ops):
    from vqacl_amd._lib import Vlt5Error
    w = ops.quant_w4(torch.randn(32, 64, generator=gen(1)).to(dev), 32)
    x = torch.zeros(2, 64, device=dev, dtype=BF)
    c = ops.kv_pages(4, 2, 64, 16, torch.int8, dev)
    t, n = ints(dev, [[0, 1], [2, 3]]), ints(dev, [3, 20])
    q = torch.zeros(2, 256, device=dev, dtype=BF)
    bad = [
        lambda: ops.quant_w4(torch.zeros(4, 48, device=dev)), lambda: ops.quant_w4(torch.zeros(4, 64, device=dev), 16), lambda: ops.quant_w4(torch.zeros(4, 64)),
        lambda: ops.quant_w4(torch.zeros(4, 64, device=dev).half()),
        lambda: ops.decode_linear_w4(x.float(), w), lambda: ops.decode_linear_w4(x[:, :32], w), lambda: ops.decode_linear_w4(x.cpu(), w),
        lambda: ops.decode_linear_w4(torch.zeros(257, 64, device=dev, dtype=BF), w), lambda: ops.decode_linear_w4(x, w._replace(scales=w.scales[:, :1].contiguous())),
        lambda: ops.decode_linear_w4(x, w, resid=torch.zeros(2, 32, device=dev, dtype=BF)), lambda: ops.decode_linear_w4(x, w, out=torch.zeros(2, 31, device=dev)),
        lambda: ops.decode_linear_w4(torch.zeros(2, 68, device=dev, dtype=BF)[:, 4:], w), lambda: ops.decode_linear_w4(x[:1].expand(2, 64), w),
        lambda: ops.kv_pages(4, 2, 64, 16, torch.float16, dev),
        lambda: ops.kv_page_write(c, q[:, :128], q[:, :64], t, n), lambda: ops.kv_page_write(c, q[:, :128].float(), q[:, :128].float(), t, n),
        lambda: ops.kv_page_write(c, q[:1, :128], q[:1, :128], t, n), lambda: ops.kv_page_write(c, q[:, :128], q[:, :128], t.long(), n),
        lambda: ops.kv_page_write(c, q[:, :128], q[:, :128], t, n, cu_q=ints(dev, [0, 1])), lambda: ops.kv_page_read(c, t, n.cpu(), 4), lambda: ops.kv_page_read(c, t[0], n, 4),
        lambda: ops.kv_page_read(c._replace(k_scale=None), t, n, 4), lambda: ops.kv_page_read(ops.kv_pages(4, 2, 96, 16, torch.int8, dev), t, n, 4),
        lambda: ops.kv_page_read(ops.kv_pages(4, 2, 64, 24, torch.int8, dev), t, n, 4), lambda: ops.kv_page_read(c._replace(v=c.v[:, :, :8]), t, n, 4),
        lambda: ops.paged_attn(q[:, :192], c, t, n), lambda: ops.paged_attn(q, c, t, n, rel_bias=torch.zeros(3, 8, device=dev)),
        lambda: ops.paged_attn(q, c, t, n, causal=False, rel_bias=torch.zeros(4, 8, device=dev)), lambda: ops.paged_attn(q, c, t, n, out=q[:1]),
        lambda: ops.paged_attn(q[:1].expand(2, 256), c, t, n), lambda: ops.paged_attn(q, c, t, n[:1]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(Vlt5Error):
            f()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()
    assert ops.paged_attn(q[:0], c, t, n, cu_q=ints(dev, [0, 0, 0])).shape == (0, 256)
    k, v = ops.kv_page_read(c, t, n, 0)
    assert k.shape == v.shape == (2, 0, 128)


# ---- the corners of a call --------------------------------------------------------------------------------------------------------
def test_decode_linear_w4_slabs_with_a_short_end(dev, ops):
    """Rows of x that do not fit LDS, of a length that is no multiple of 128 or of the group; extreme values beside zeros."""
    for rows, N, K, group, split in ((16, 40, 11040, 128, True), (13, 17, 9952, 64, True), (40, 100, 4640, 32, True), (16, 4400, 5088, 64, False), (16, 4112, 5152, 64, True), (30, 1000, 10016, 128, True), (100, 700, 5024, 32, False)):
        from vqacl_amd._lib import lib
        assert (lib().vlt5_decode_linear_w4_workspace_bytes(rows, N, K) > 0) == split      # slabs in workgroups of their own, or one after the other
        g = gen(K)
        w = ops.quant_w4((torch.randn(N, K, generator=g) * K ** -0.5).to(dev), group)
        x = torch.randn(rows, K, generator=g).to(BF)
        x[0] = 0
        x[1, ::7] *= 1e4
        v = w4_value(w)
        y = ops.decode_linear_w4(x.to(dev), w, out_f32=True).cpu().double()
        ref = x.double() @ v.t()
        acc = (group + -(-K // group) + 16) * U * (x.double().abs() @ v.abs().t())
        assert bool(((y - ref).abs() <= acc).all())
        assert bool((y[0] == 0).all())
        resid = torch.randn(rows, N, generator=g).to(dev)
        z = ops.decode_linear_w4(x.to(dev), w, alpha=0.5, relu=True, resid=resid, out=resid.to(BF)).cpu().double()
        want = (0.5 * ref + resid.cpu().double()).clamp_min(0)
        assert bool(((z - want).abs() <= acc + U * want + H * want).all())


@pytest.mark.parametrize("rows,N,K,group", [(256, 1100, 7712, 64), (250, 2100, 4128, 32), (129, 2053, 8224, 128), (241, 9001, 992, 128), (255, 8452, 1024, 32)])
def test_decode_linear_w4_many_rows(dev, ops, rows, N, K, group):
    """More than 2^31 multiply-adds: 32 rows a workgroup, split and not, ends inside a chunk and inside a group, rows and columns past the last tile."""
    from vqacl_amd._lib import lib
    assert rows * N * K > 2 ** 31 and (lib().vlt5_decode_linear_w4_workspace_bytes(rows, N, K) > 0) == (K >= 4096)
    g = gen(rows + N)
    w = ops.quant_w4((torch.randn(N, K, generator=g) * K ** -0.5).to(dev), group)
    wide = torch.full((rows, K + 8), float("nan")).to(BF)
    x = wide[:, :K]
    x.copy_(torch.randn(rows, K, generator=g))
    x[2] = 0
    v, xd = w4_value(w), wide.to(dev)[:, :K]
    ref = x.double() @ v.t()
    acc = (group + -(-K // group) + 16) * U * (x.double().abs() @ v.abs().t())
    y = ops.decode_linear_w4(xd, w, out_f32=True).cpu().double()
    assert bool(((y - ref).abs() <= acc).all()) and bool((y[2] == 0).all())
    resid = torch.randn(rows, N, generator=g)
    room = torch.full((rows + 2, N + 3), 7.0, device=dev, dtype=BF)
    ops.decode_linear_w4(xd, w, alpha=-2.0, relu=True, resid=resid.to(dev), out=room[1:-1, :N])
    want = (-2 * ref + resid.double()).clamp_min(0)
    assert bool(((room[1:-1, :N].cpu().double() - want).abs() <= 2 * acc + U * want + H * want).all())
    room[1:-1, :N] = 7
    assert bool((room == 7).all())


@pytest.mark.parametrize("kind", KINDS)
def test_more_new_tokens_than_keys(dev, ops, kind):
    """Positions below zero: nothing is written for them, they see nothing; the others are as ever."""
    lens, new = [3, 40], [7, 2]
    c, table = make_cache(ops, dev, [16, 48], 2, 64, 16, kind, seed=31)
    before = [None if t is None else raw(t).cpu().clone() for t in c]
    x = torch.randn(9, 128, generator=gen(3)).to(BF).to(dev)
    args = (table.to(dev), ints(dev, lens))
    ops.kv_page_write(c, x, x, *args, cu_q=ints(dev, starts(new)))
    codes, sc = plain_codes(x.cpu().view(9, 2, 64), kind)
    p = int(table[0, 0])
    assert torch.equal(raw(c.k)[p, :, :3].cpu(), raw(codes)[4:7].transpose(0, 1)) and torch.equal(raw(c.k)[p, :, 3:].cpu(), before[0][p, :, 3:])
    out, lse = ops.paged_attn(x, c, *args, cu_q=ints(dev, starts(new)), want_lse=True)
    assert bool((out[:4] == 0).all()) and bool((lse[:4] == -math.inf).all())
    ref, tol, _ = attn_ref(x[4:].cpu(), c, table, [3, 2], lens, 2, 1.0, True, None)
    assert bool(((out[4:].cpu().double().view(5, 2, 64) - ref).abs() <= tol).all())


@pytest.mark.parametrize("new", [[3, 9], [90, 40]])
def test_max_q_limits_what_is_processed(dev, ops, new):
    """Tokens past max_q are left alone by the write and by the attention."""
    lens = [100, 60]
    c, table = make_cache(ops, dev, lens, 2, 64, 16, torch.int8, seed=32)
    n, most = sum(new), min(new)
    x = torch.randn(n, 128, generator=gen(4)).to(BF).to(dev)
    args = (table.to(dev), ints(dev, lens))
    full = ops.paged_attn(x, c, *args, cu_q=ints(dev, starts(new)))
    out = torch.full((n, 128), 3.0, device=dev, dtype=BF)
    ops.paged_attn(x, c, *args, cu_q=ints(dev, starts(new)), max_q=most, out=out)
    for b in range(2):
        s = starts(new)[b]
        assert bool((out[s + most: s + new[b]] == 3.0).all())
        ref, tol, _ = attn_ref(x.cpu(), c, table, new, lens, 2, 1.0, True, None)
        err = (out[s: s + most].cpu().double().view(-1, 2, 64) - ref[s: s + most]).abs()
        assert bool((err <= tol[s: s + most]).all())
    assert full.shape == out.shape
    before = raw(c.k).clone()
    ops.kv_page_write(c, x, x, *args, cu_q=ints(dev, starts(new)), max_q=1)
    changed = (raw(c.k) != before).any(-1).nonzero().cpu()
    want = {(int(table[b, (lens[b] - new[b]) // 16]), (lens[b] - new[b]) % 16) for b in range(2)}
    assert {(int(p), int(r)) for p, _, r in changed} == want


def test_strided_rows_and_shared_pages(dev, ops):
    """q, k, v and out as slices of wider buffers; two sequences that share the pages of a prefix; out in the place of q."""
    c, _ = make_cache(ops, dev, [96, 96], 2, 64, 16, FP8, seed=33)
    table = torch.tensor([[0, 1, 2, 3], [0, 1, 4, 5]], dtype=torch.int32)                  # 32 positions in common
    lens, new = [50, 60], [5, 20]
    wide = torch.randn(25, 904, generator=gen(5)).to(BF).to(dev)
    q, k, v = wide[:, 8:264], wide[:, 264:392], wide[:, 400:528]
    args = (table.to(dev), ints(dev, lens))
    ops.kv_page_write(c, k, v, *args, cu_q=ints(dev, starts(new)))
    kr, _ = ops.kv_page_read(c, *args, 64)
    kk, _ = held(c, table, 1, 60)
    assert torch.equal(kr[1, :60].cpu().double(), kk.flatten(1).float().to(BF).double()) and torch.equal(kr[0, :32], kr[1, :32])
    buf = torch.full((25, 304), 2.0, device=dev, dtype=BF)
    out = ops.paged_attn(q, c, *args, cu_q=ints(dev, starts(new)), out=buf[:, 16:272])
    ref, tol, _ = attn_ref(q.cpu(), c, table, new, lens, 4, 1.0, True, None)
    assert bool(((out.cpu().double().view(25, 4, 64) - ref).abs() <= tol).all())
    assert bool((buf[:, :16] == 2).all()) and bool((buf[:, 272:] == 2).all())
    mine = q.contiguous()
    assert torch.equal(ops.paged_attn(mine, c, *args, cu_q=ints(dev, starts(new)), out=mine), out) and torch.equal(mine, out)
    from vqacl_amd._lib import Vlt5Error
    for bad in (lambda: ops.paged_attn(wide[:, 4:260], c, *args, cu_q=ints(dev, starts(new))), lambda: ops.kv_page_write(c, wide[:, 4:132], v, *args, cu_q=ints(dev, starts(new))),
                lambda: ops.paged_attn(q, c, *args, cu_q=ints(dev, starts(new)), scale=0.0), lambda: ops.paged_attn(q, c, *args, cu_q=ints(dev, starts(new)), scale=-1.0)):
        with pytest.raises(Vlt5Error):
            bad()


@pytest.mark.parametrize("scale", [1e-39, 1e-30, 30.0])
@pytest.mark.parametrize("new", [1, 40])
def test_extreme_scales(dev, ops, scale, new):
    """All keys alike, and one key alone: the running maximum's slack follows the scale."""
    lens = [300]
    c, table = make_cache(ops, dev, lens, 2, 64, 16, torch.int8, seed=34)
    check_attn(ops, dev, c, table, [new], lens, 4, scale=scale, seed=1)


@pytest.mark.parametrize("kind", [torch.int8, FP8])
def test_a_token_that_is_not_finite_is_seen_by_later_ones_only(dev, ops, kind):
    """8-bit types: a NaN or an infinity in a new token's key or value shows in the tokens that see it and in no other."""
    new, lens = [70], [90]
    c, table = make_cache(ops, dev, lens, 1, 64, 16, kind, seed=35)
    x = torch.randn(70, 64, generator=gen(6)).to(BF)
    x[41, 5], x[41, 6] = math.nan, math.inf
    for k, v in ((x, x.nan_to_num(0, 0, 0)), (x.nan_to_num(0, 0, 0), x)):
        ops.kv_page_write(c, k.to(dev), v.to(dev), table.to(dev), ints(dev, lens), cu_q=ints(dev, [0, 70]))
        for heads in (1, 4):                                                               # through both kernels
            out = ops.paged_attn(torch.ones(70, 64 * heads, device=dev, dtype=BF), c, table.to(dev), ints(dev, lens), cu_q=ints(dev, [0, 70]), scale=0.1)
            assert bool(torch.isfinite(out[:41]).all()) and bool(torch.isnan(out[41:]).all())


def test_a_cold_call_inside_a_capture_and_two_graphs(dev, ops):
    """Two graphs of the same step, replayed in turn and with eager calls between: each has a workspace of its own."""
    lens = [6000]
    c, table = make_cache(ops, dev, lens, 4, 128, 64, FP8, seed=36)
    t, n = table.to(dev), ints(dev, lens)
    qs = [torch.randn(1, 16 * 128, generator=gen(50 + i)).to(BF).to(dev) for i in range(3)]
    want = [ops.paged_attn(q, c, t, n, scale=0.09) for q in qs]
    graphs = []
    for q in qs[:2]:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.paged_attn(q, c, t, n, scale=0.09)
        graphs.append((g, y))
    for i in (0, 1, 1, 0, 1):
        graphs[i][0].replay()
        assert torch.equal(ops.paged_attn(qs[2], c, t, n, scale=0.09), want[2])
        torch.cuda.synchronize()
        assert torch.equal(graphs[i][1], want[i])


def test_no_factor_and_no_sequences(dev, ops):
    from vqacl_amd._lib import Vlt5Error
    w = ops.quant_w4(torch.randn(8, 64, generator=gen(1)).to(dev), 32)
    with pytest.raises(Vlt5Error):
        ops.decode_linear_w4(torch.zeros(1, 64, device=dev, dtype=torch.bfloat16), w, alpha=0.0)
    none = torch.zeros(0, 3, device=dev, dtype=torch.int32)
    c = ops.kv_pages(2, 1, 64, 16, torch.int8, dev)
    k, v = ops.kv_page_read(c, none, none[:, 0].contiguous(), 5)
    assert k.shape == v.shape == (0, 5, 64)
    x = torch.zeros(0, 64, device=dev, dtype=torch.bfloat16)
    ops.kv_page_write(c, x, x, none, none[:, 0].contiguous())
    assert ops.paged_attn(x, c, none, none[:, 0].contiguous()).shape == (0, 64)


@pytest.mark.parametrize("alpha", [1e-50, -1e-50, 2.0 ** -150, -0.0])
def test_a_factor_that_is_zero_in_f32_is_refused(dev, ops, alpha):
    """The descriptor holds alpha in f32, where 0 stands for 1."""
    from vqacl_amd._lib import Vlt5Error
    w = ops.quant_w4(torch.randn(8, 64, generator=gen(1)).to(dev), 32)
    x = torch.ones(1, 64, device=dev, dtype=BF)
    with pytest.raises(Vlt5Error):
        ops.decode_linear_w4(x, w, alpha=alpha)
    small = 2.0 ** -100                                                                     # an f32 number: a factor as any other
    assert torch.equal(ops.decode_linear_w4(x, w, alpha=small, out_f32=True), small * ops.decode_linear_w4(x, w, out_f32=True))


@pytest.mark.parametrize("rows,N,K,group,runs", [(5, 4300, 14112, 64, 3), (6, 5000, 12320, 128, 3), (62, 4600, 5088, 32, 3), (50, 5400, 6176, 64, 4), (63, 5000, 5088, 128, 3)])
def test_decode_linear_w4_split_on_a_chip_that_is_not_full(dev, ops, rows, N, K, group, runs):
    """Runs on both sides of two workgroups a CU, with ends inside a chunk, a group and a tile."""
    from vqacl_amd._lib import lib
    assert lib().vlt5_decode_linear_w4_workspace_bytes(rows, N, K) == 4 * rows * N * runs
    g = gen(rows + K)
    w = ops.quant_w4((torch.randn(N, K, generator=g) * K ** -0.5).to(dev), group)
    x = torch.randn(rows, K, generator=g).to(BF)
    v = w4_value(w)
    ref = x.double() @ v.t()
    acc = (group + -(-K // group) + 16) * U * (x.double().abs() @ v.abs().t())
    y = ops.decode_linear_w4(x.to(dev), w, out_f32=True).cpu().double()
    assert bool(((y - ref).abs() <= acc).all())


def test_decode_linear_w4_outputs_beside_their_inputs(dev, ops):
    """Slices of one buffer that share no element are taken, whatever their order; those that do are refused."""
    from vqacl_amd._lib import Vlt5Error
    w = ops.quant_w4(torch.randn(64, 64, generator=gen(1)).to(dev), 32)
    first = torch.randn(20, 192, generator=gen(2)).to(BF).to(dev)
    for rows in (1, 20):
        for a, b in ((0, 64), (64, 0), (0, 128), (128, 64), (56, 120)):
            buf = first.clone()
            want = ops.decode_linear_w4(buf[:rows, a:a + 64].clone(), w)
            got = ops.decode_linear_w4(buf[:rows, a:a + 64], w, out=buf[:rows, b:b + 64])
            assert torch.equal(got, want) and torch.equal(buf[:rows, a:a + 64], first[:rows, a:a + 64])
        for a, b in ((0, 0), (0, 56), (64, 8)):
            buf = first.clone()
            with pytest.raises(Vlt5Error):
                ops.decode_linear_w4(buf[:rows, a:a + 64], w, out=buf[:rows, b:b + 64])
    above = first.clone()
    assert torch.equal(ops.decode_linear_w4(above[1:3, :64], w, out=above[4:6, 64:128]), ops.decode_linear_w4(first[1:3, :64], w))
    two = torch.randn(6, 64, generator=gen(3)).to(dev)
    want = ops.decode_linear_w4(first[:3, :64], w, resid=two[:3].clone(), out_f32=True)
    assert torch.equal(ops.decode_linear_w4(first[:3, :64], w, resid=two[:3], out=two[3:]), want)
    with pytest.raises(Vlt5Error):
        ops.decode_linear_w4(first[:3, :64], w, resid=two[:3], out=two[1:4])


@pytest.mark.parametrize("new,lens", [([1, 1, 1], [50, 3000, 7]), ([3, 80, 20], [50, 300, 20]), ([150], [2000])])
def test_attention_in_the_place_of_its_queries(dev, ops, new, lens):
    """`out` beside q in one buffer and as q itself, single tokens and chunks, split and not; over q in any other way it is refused."""
    from vqacl_amd._lib import Vlt5Error
    c, table = make_cache(ops, dev, lens, 2, 64, 16, torch.int8, seed=37)
    n, args, kw = sum(new), (table.to(dev), ints(dev, lens)), dict(cu_q=ints(dev, starts(new)), max_q=max(new), scale=0.1)
    first = torch.randn(n, 768, generator=gen(6)).to(BF).to(dev)
    want = ops.paged_attn(first[:, 128:384].contiguous(), c, *args, **kw)
    for a, b in ((128, 384), (128, 128), (512, 0)):
        buf = first.clone()
        buf[:, a:a + 256] = first[:, 128:384]
        assert torch.equal(ops.paged_attn(buf[:, a:a + 256], c, *args, out=buf[:, b:b + 256], **kw), want)
    with pytest.raises(Vlt5Error):
        ops.paged_attn(first[:, :256], c, *args, out=first[:, 64:320], **kw)
    if n > 1:
        flat = torch.zeros(n + 1, 256, device=dev, dtype=BF)
        with pytest.raises(Vlt5Error):
            ops.paged_attn(flat[:n], c, *args, out=flat[1:], **kw)


@pytest.mark.parametrize("max_kv", [-3, 1, 900, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("lens", [[600], [1500]])
def test_any_max_kv_is_taken(dev, ops, max_kv, lens):
    """Shorter and longer than the table, which is what a sequence can have: a hint for the split."""
    c, table = make_cache(ops, dev, lens, 2, 64, 16, FP8, seed=38)
    for new in ([1], [50]):
        check_attn(ops, dev, c, table, new, lens, 4, max_kv=max_kv, seed=1)


@pytest.mark.parametrize("kind", [BF, FP8])
@pytest.mark.parametrize("d,g,new,lens,nd", [
    (64, 1, [20], [50], 0), (128, 3, [21, 9], [40, 70], 0), (64, 2, [70], [90], 40), (128, 1, [130], [330], 0), (64, 4, [150, 60], [150, 300], 0), (128, 4, [40], [2600], 16), (64, 16, [4], [1500], 0), (128, 3, [5], [29], 0), (64, 40, [4], [60], 0),
    (64, 1, [131] * 66, [131 + 3 * b for b in range(66)], 0), (64, 1, [131] * 66, [131 + 3 * b for b in range(66)], 30), (128, 1, [131] * 66, [131 + 3 * b for b in range(66)], 0),
])
def test_a_value_that_is_not_finite_is_seen_by_later_tokens_only(dev, ops, kind, d, g, new, lens, nd):
    """Values of the cache that are infinite or NaN (e4m3: NaN) show in their column, in the tokens that see them, and nowhere else."""
    hk = 2
    c, table = make_cache(ops, dev, lens, hk, d, 16, kind, seed=d + g)
    n = sum(new)
    q = torch.randn(n, hk * g * d, generator=gen(n)).to(BF).to(dev)
    bias = None if not nd else torch.randn(hk * g, nd, generator=gen(nd)).to(dev)
    args, kw = (table.to(dev), ints(dev, lens)), dict(cu_q=ints(dev, starts(new)), max_q=max(new), scale=0.1, rel_bias=bias)
    clean, lse = ops.paged_attn(q, c, *args, want_lse=True, **kw)
    want = clean.float().view(n, hk, g, d).clone()
    marks = []                                                                              # sequence, position, head, column, value
    for b in range(len(new)):
        p0 = lens[b] - new[b]
        marks += [(b, p0 + new[b] // 2, 0, 5, math.nan), (b, p0 + new[b] // 3, 1, d - 1, math.inf), (b, p0 + new[b] // 3, 1, 7, math.inf), (b, lens[b] - 1, 1, 7, -math.inf),
                  (b, p0 + 1, 0, 0, -math.inf), (b, lens[b] - 2, 0, d // 2, math.inf)]
    for b, pos, h, col, x in marks:
        p, r = int(table[b, pos // 16]), pos % 16
        if kind == BF:
            c.v[p, h, r, col] = x
        else:
            raw(c.v)[p, h, r, col] = 0x7f if x > 0 else 0xff
            x = math.nan
        seen = slice(starts(new)[b] + pos - (lens[b] - new[b]), starts(new)[b + 1])
        want[seen, h, :, col] = want[seen, h, :, col].masked_fill(torch.isfinite(want[seen, h, :, col]), 0) + x
    for _ in range(2):
        got, l2 = ops.paged_attn(q, c, *args, want_lse=True, **kw)
        got = got.float().view(n, hk, g, d)
        wrong = int((torch.isnan(got) != torch.isnan(want)).sum()), int((torch.isinf(got) != torch.isinf(want)).sum()), int((l2 != lse).sum())
        assert wrong == (0, 0, 0)
        odd = ~torch.isfinite(want)
        assert torch.equal(got.masked_fill(odd, 0), want.masked_fill(odd, 0))                # the rest as without them
        assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    assert bool(torch.isnan(want).any()) and (kind == FP8 or bool(torch.isinf(want).any()))


@pytest.mark.parametrize("kind", KINDS)
def test_the_first_of_several_tokens_does_not_see_the_others(dev, ops, kind):
    """max_q = 1: the one token that is processed is not the sequence's last, and what the others left is not its."""
    lens, new = [40, 70], [3, 9]
    c, table = make_cache(ops, dev, lens, 2, 64, 16, kind, seed=41)
    q = torch.randn(12, 512, generator=gen(8)).to(BF).to(dev)
    args, kw = (table.to(dev), ints(dev, lens)), dict(cu_q=ints(dev, [0, 3, 12]), scale=0.1)
    want = ops.paged_attn(q, c, *args, **kw)[[0, 3]]
    for b in range(2):
        for pos in range(lens[b] - new[b] + 1, lens[b]):
            p, r = int(table[b, pos // 16]), pos % 16
            for pages, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
                raw(pages)[p, :, r] = math.nan if kind == BF else 127
                if scales is not None:
                    scales[p, :, r] = math.nan
    got = ops.paged_attn(q, c, *args, max_q=1, **kw)[[0, 3]]
    assert torch.equal(got, want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal,g,nd", [(True, 1, 0), (True, 1, 40), (True, 2, 300), (False, 1, 0)])
def test_chunks_on_a_full_chip(dev, ops, kind, d, causal, g, nd):
    """More tiles of 128 rows than CUs: four waves a workgroup, which read all of its keys; two row tiles a sequence, one sequence whose page ids
    are loaded twice (more than 16 tiles of 64 keys), one with a page that is not there, one that is empty and one with one token."""
    B, hk = 17, 8
    news = [140 - 4 * b for b in range(B)]
    lens = [n + (31 * b) % 90 for b, n in enumerate(news)]
    lens[2] = 1150
    news[5] = lens[5] = 0
    news[6] = 1
    c, table = make_cache(ops, dev, lens, hk, d, 16, kind, seed=d + nd)
    table[9, 3] = -1
    assert -(-max(news) * g // 128) * B * hk > 256
    bias = 2 * torch.randn(hk * g, nd, generator=gen(nd)) if nd else None
    check_attn(ops, dev, c, table, news, lens, hk * g, causal=causal, bias=bias, seed=1)


@pytest.mark.parametrize("g,nd", [(8, 64), (8, 65), (8, 128), (8, 129), (2, 512), (2, 513), (2, 832), (2, 833), (4, 256), (4, 257), (4, 320), (4, 321), (1, 1024), (1, 1025), (1, 1856), (1, 1857)])
@pytest.mark.parametrize("new", [[1, 1], [5, 2], [90, 33]])
def test_bias_tables_that_fit_lds_and_that_do_not(dev, ops, g, nd, new):
    """Both sides of what either kernel keeps in LDS (1024 entries; 2048 with 192 of padding a head), contexts longer and shorter than the table."""
    kind, d = KINDS[(g + nd + len(new) + new[0]) % 3], 64 if (nd + new[0]) % 4 < 2 else 128
    lens = [nd + 150, max(new[1], min(nd // 2, 400))]
    c, table = make_cache(ops, dev, lens, 2, d, 32, kind, seed=nd)
    check_attn(ops, dev, c, table, new, lens, 2 * g, bias=2 * torch.randn(2 * g, nd, generator=gen(nd)), seed=1)
