"""Cases of the low-precision token-step: products with 4-bit weights, the paged key/value cache, and the attention that reads it.

  w4    out[m, n] = act(sum_k x[m, k] * value(code[n, k]) * scale[n, k // group] (+ resid[m, n])): few rows against a weight whose 4-bit
        codes are e2m1 numbers (sign, two exponent bits, one mantissa bit), one bf16 scale for every `group` consecutive k
  kv    new keys | values go into the pages of the cache (int8 or e4m3 codes with one f32 scale per token and head: the largest
        magnitude / 127 or / 448; or bf16 as they are), then the whole context of every sequence is read back as bf16
  attn  softmax(scale * q K^T + bias) V for the newest tokens of every sequence over its pages: one token each, or a chunk of them

A sequence's position p lives in row p % page of page table[b, p // page]; pages are [number, kv head, row, d_kv].  Token i of a sequence
with n new tokens stands at position kv_len - n + i; the new tokens of all sequences lie behind one another (cu_q: first token of each).
"""
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def listed():
    return [
        # one sequence, one token: an attention output projection of the base model (latency counts)
        dict(name="w4_one_row", op="w4", rows=1, n=768, k=768, group=32, relu=False, resid=False),
        # the q | k | v projection of a token-step at the batch the framework decodes with
        dict(name="w4_qkv_80", op="w4", rows=80, n=2304, k=768, group=64, relu=False, resid=False),
        # the vocabulary projection for a small batch
        dict(name="w4_vocab_16", op="w4", rows=16, n=32200, k=768, group=128, relu=False, resid=False),
        # the second FFN product of a large model for a few sequences, added to the f32 residual stream; an odd number of columns
        dict(name="w4_down_5", op="w4", rows=5, n=4097, k=14336, group=64, relu=False, resid=True),
        # encoder-side keys | values of the evaluation batch, written once, read back for the dense cross-attention
        dict(name="kv_memory_80", op="kv", batch=80, old=0, new=58, heads=12, d=64, page=64, cache="int8", ragged=True),
        # chunks of long prompts of a grouped-head model behind what the cache holds already
        dict(name="kv_prompt_4", op="kv", batch=4, old=3000, new=1000, heads=8, d=128, page=32, cache="fp8", ragged=True),
        # cross-attention of a token-step: every key of the encoder's memory is visible
        dict(name="attn_cross_80", op="attn", batch=80, q=1, kv=58, heads=12, kv_heads=12, d=64, page=64, cache="int8", causal=False, bias=0, ragged=True),
        # decoder self-attention of a token-step with the relative-position bias, ragged answers
        dict(name="attn_self_100", op="attn", batch=100, q=1, kv=500, heads=12, kv_heads=12, d=64, page=16, cache="fp8", causal=True, bias=128, ragged=True),
        # one sequence with a long context: the keys have to be split
        dict(name="attn_one_long", op="attn", batch=1, q=1, kv=131071, heads=32, kv_heads=8, d=128, page=64, cache="int8", causal=True, bias=0, ragged=False),
        # the throughput of single tokens over long caches
        dict(name="attn_token_32", op="attn", batch=32, q=1, kv=16384, heads=32, kv_heads=8, d=128, page=128, cache="fp8", causal=True, bias=0, ragged=True),
        # a chunk of a prompt with the relative-position bias
        dict(name="attn_chunk_bias_8", op="attn", batch=8, q=200, kv=712, heads=12, kv_heads=12, d=64, page=64, cache="int8", causal=True, bias=128, ragged=True),
        # a long chunk over a long bf16 cache: matrix products
        dict(name="attn_chunk_1", op="attn", batch=1, q=2048, kv=16384, heads=32, kv_heads=8, d=128, page=64, cache="bf16", causal=True, bias=0, ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("w4", "kv", "attn", "attn"))
    while True:
        if op == "w4":
            c = dict(op="w4", rows=_log(rng, 1, 256), n=_log(rng, 64, 33000), k=32 * _log(rng, 2, 512), group=rng.choice((32, 64, 128)),
                     relu=rng.random() < 0.3, resid=rng.random() < 0.3)
            if c["rows"] * c["n"] * c["k"] > 16 * 32200 * 768 * 3:
                continue
        elif op == "kv":
            c = dict(op="kv", batch=_log(rng, 1, 100), old=rng.choice((0, _log(rng, 1, 4000))), new=_log(rng, 1, 1500), heads=rng.choice((4, 8, 12, 16)),
                     d=rng.choice((64, 128)), page=rng.choice((16, 32, 64, 128)), cache=rng.choice(("int8", "fp8", "bf16")), ragged=rng.random() < 0.8)
            if c["batch"] * (c["old"] + c["new"]) * c["heads"] * c["d"] > 4 * 4000 * 8 * 128:
                continue
        else:
            kv_heads = rng.choice((2, 4, 8, 12))
            q = rng.choice((1, 1, _log(rng, 2, 64), _log(rng, 64, 2000)))
            kv = max(q, _log(rng, 8, 60000))
            c = dict(op="attn", batch=_log(rng, 1, 100), q=q, kv=kv, heads=kv_heads * rng.choice((1, 1, 2, 3, 4, 8)), kv_heads=kv_heads, d=rng.choice((64, 128)),
                     page=rng.choice((16, 32, 64, 128)), cache=rng.choice(("int8", "fp8", "bf16")), causal=rng.random() < 0.8, bias=rng.choice((0, 0, 32, 128)),
                     ragged=rng.random() < 0.8)
            if not c["causal"]:
                c["bias"] = 0
            if c["batch"] * kv * kv_heads * c["d"] > 32 * 16384 * 8 * 128 or c["batch"] * q * kv * c["heads"] * c["d"] > 2048 * 16384 * 32 * 128:
                continue
            if c["batch"] * q * kv * c["heads"] > 2048 * 16384 * 32:
                continue
        return c


def _lengths(most, least, batch, ragged):
    """Lengths between `least` and `most`, a function of the case alone; the first sequence has the longest."""
    if not ragged:
        return [most] * batch
    return [most - (b * 7919 * (most - least + 3) // 10007) % (most - least + 1) for b in range(batch)]


def _shape(c):
    """(new tokens, context lengths) of every sequence."""
    if c["op"] == "kv":
        new = _lengths(c["new"], (c["new"] + 1) // 2, c["batch"], c["ragged"])
        old = _lengths(c["old"], c["old"] // 2, c["batch"], c["ragged"])
        return new, [a + b for a, b in zip(new, old)]
    new = _lengths(c["q"], (c["q"] + 1) // 2, c["batch"], c["ragged"])
    return new, [max(a, b) for a, b in zip(new, _lengths(c["kv"], (c["kv"] + 1) // 2, c["batch"], c["ragged"]))]


def _quantise(x, kind):
    """x f32 [..., d] -> (codes, scale f32 [...])."""
    if kind == "bf16":
        return x.to(BF16), None
    most = 127.0 if kind == "int8" else 448.0
    scale = x.abs().amax(-1) / most
    y = torch.where(scale.unsqueeze(-1) > 0, x / scale.unsqueeze(-1), torch.zeros_like(x)).clamp(-most, most)
    return (torch.round(y).to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)), scale


def _keys(g, dev, *shape):
    """Keys and values as a projection leaves them: some channels are several times larger than others."""
    gain = torch.exp(0.5 * torch.randn(shape[-1], device=dev, generator=g))
    return (torch.randn(*shape, device=dev, generator=g) * gain).to(BF16)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    c = case
    if c["op"] == "w4":
        w = torch.randn(c["n"], c["k"], device=dev, generator=g) * c["k"] ** -0.5
        groups = -(-c["k"] // c["group"])
        pad = torch.nn.functional.pad(w, (0, groups * c["group"] - c["k"])).view(c["n"], groups, c["group"])
        scales = (pad.abs().amax(-1) / 6.0).to(BF16)
        y = (pad / scales.float().clamp_min(1e-30).unsqueeze(-1)).view(c["n"], -1)[:, : c["k"]].contiguous()
        del w, pad
        mag = torch.bucketize(y.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=dev)).to(torch.uint8)
        code = mag | ((y < 0).to(torch.uint8) << 3)
        codes = code[:, 0::2] | (code[:, 1::2] << 4)          # byte j of a row: k = 2j in the low four bits, 2j + 1 in the high ones
        x = torch.randn(c["rows"], c["k"], device=dev, generator=g).to(BF16)
        resid = torch.randn(c["rows"], c["n"], device=dev, generator=g) if c["resid"] else None
        return dict(c=c, x=x, codes=codes.contiguous(), scales=scales, resid=resid)
    new, lens = _shape(c)
    B, d, page = c["batch"], c["d"], c["page"]
    Hk = c["heads"] if c["op"] == "kv" else c["kv_heads"]
    per = -(-max(lens) // page)
    used = [-(-n // page) for n in lens]
    pages = sum(used) + 3
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    at = torch.tensor([sum(used[:b]) for b in range(B)], device=dev).unsqueeze(1) + torch.arange(per, device=dev)
    table = torch.where(torch.arange(per, device=dev) < torch.tensor(used, device=dev).unsqueeze(1), order[at.clamp_max(pages - 1)], order[-1]).to(torch.int32)
    k, ks = _quantise(_keys(g, dev, pages, Hk, page, d).float(), c["cache"])
    v, vs = _quantise(_keys(g, dev, pages, Hk, page, d).float(), c["cache"])
    total = sum(new)
    ints = dict(device=dev, dtype=torch.int32)
    cu = torch.tensor([sum(new[:b]) for b in range(B + 1)], **ints)
    which = torch.repeat_interleave(torch.arange(B, device=dev), torch.tensor(new, device=dev))
    s = dict(c=c, k=k, v=v, ks=ks, vs=vs, table=table, lens=torch.tensor(lens, **ints), cu=cu, new=max(new), most=max(lens),
             tok_b=which, tok_i=torch.arange(total, device=dev) - cu[which].long())          # sequence and place of every new token
    if c["op"] == "kv":
        both = _keys(g, dev, total, 2 * Hk * d)
        s["new_k"], s["new_v"] = both[:, : Hk * d], both[:, Hk * d:]
        return s
    H = c["heads"]
    qkv = torch.randn(total, (H + 2 * Hk) * d, device=dev, generator=g)
    s["scale"] = 1.0 if c["bias"] or not c["causal"] else d ** -0.5          # T5 does not scale its scores
    s["q"] = (qkv * (d ** -0.5 / s["scale"])).to(BF16)[:, : H * d]
    s["bias"] = torch.randn(H, c["bias"], device=dev, generator=g) if c["bias"] else None
    return s


def _own(s):
    from vqacl_amd import ops
    c = s["c"]
    if c["op"] == "w4":
        w = ops.W4Weight(s["codes"], s["scales"], c["group"])
        return ops.decode_linear_w4(s["x"], w, relu=c["relu"], resid=s["resid"], out_f32=c["resid"])
    cache = ops.KVPages(s["k"], s["v"], s["ks"], s["vs"])
    if c["op"] == "kv":
        ops.kv_page_write(cache, s["new_k"], s["new_v"], s["table"], s["lens"], cu_q=s["cu"], max_q=s["new"])
        return ops.kv_page_read(cache, s["table"], s["lens"], s["most"])
    cu = None if c["q"] == 1 else s["cu"]
    return ops.paged_attn(s["q"], cache, s["table"], s["lens"], cu_q=cu, max_q=s["new"], max_kv=s["most"], scale=s["scale"], causal=c["causal"], rel_bias=s["bias"])


def _context(pages, scales, table):
    """The rows of every sequence's pages, one behind the other: f32 [B, heads, rows, d]."""
    x = pages.view(torch.uint8)[table.long()].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[table.long()]
    x = x.float()
    if scales is not None:
        x = x * scales[table.long()].unsqueeze(-1)
    return x.transpose(1, 2).flatten(2, 3)


def run(state):
    if own:
        return _own(state)
    s, c = state, state["c"]
    if c["op"] == "w4":
        both = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).flatten(1)
        w = torch.tensor(E2M1, device=both.device)[both.long()]
        w = w * s["scales"].float().repeat_interleave(c["group"], 1)[:, : c["k"]]
        out = torch.matmul(s["x"].float(), w.t())
        if c["resid"]:
            out = out + s["resid"]
        if c["relu"]:
            out = out.clamp_min(0)
        return out if c["resid"] else out.to(BF16)
    lens = s["lens"].long()
    start = lens - (s["cu"][1:] - s["cu"][:-1]).long()
    pos = start[s["tok_b"]] + s["tok_i"]                       # position of every new token
    page, d = c["page"], c["d"]
    if c["op"] == "kv":
        where, row = s["table"].long()[s["tok_b"], pos // page], pos % page
        back = []
        for pages, scales, x in ((s["k"], s["ks"], s["new_k"]), (s["v"], s["vs"], s["new_v"])):
            codes, scale = _quantise(x.float().view(-1, c["heads"], d), c["cache"])
            raw = pages.view(torch.uint8) if pages.dtype == torch.float8_e4m3fn else pages
            raw[where, :, row] = codes.view(raw.dtype)
            if scale is not None:
                scales[where, :, row] = scale
            y = _context(pages, scales, s["table"])[:, :, : s["most"]]
            y = torch.where((torch.arange(s["most"], device=y.device) < lens.unsqueeze(1))[:, None, :, None], y, 0.0)
            back.append(y.transpose(1, 2).flatten(2).to(BF16))
        return tuple(back)
    B, H, Hk = c["batch"], c["heads"], c["kv_heads"]
    k, v = _context(s["k"], s["ks"], s["table"]), _context(s["v"], s["vs"], s["table"])
    q = torch.zeros(B, s["new"], H * d, device=k.device)
    q[s["tok_b"], s["tok_i"]] = s["q"].float()
    q = q.view(B, s["new"], Hk, H // Hk, d).permute(0, 2, 3, 1, 4).flatten(2, 3)               # [B, Hk, heads of the group x tokens, d]
    score = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).view(B, H, s["new"], -1)
    j = torch.arange(score.shape[-1], device=k.device)
    far = (start.unsqueeze(1) + torch.arange(s["new"], device=k.device)).unsqueeze(-1) - j    # how far a key lies behind its query
    if s["bias"] is not None:
        score = score + s["bias"][:, far.clamp(0, s["bias"].shape[1] - 1)].transpose(0, 1)
    seen = (j < lens[:, None, None]) & ((far >= 0) if c["causal"] else True)
    score = score.masked_fill(~seen.unsqueeze(1), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, Hk, -1, p.shape[-1]), v).view(B, H, s["new"], d) / torch.where(total > 0, total, 1.0)
    return out.transpose(1, 2)[s["tok_b"], s["tok_i"]].flatten(1).to(BF16)


def work(case):
    c = case
    if c["op"] == "w4":
        out = c["rows"] * c["n"] * (8 if c["resid"] else 2)
        groups = -(-c["k"] // c["group"])
        return {"bytes": c["n"] * c["k"] // 2 + 2 * c["n"] * groups + 2 * c["rows"] * c["k"] + out, "flops": 2 * c["rows"] * c["n"] * c["k"]}
    new, lens = _shape(c)
    width = 2 if c["cache"] == "bf16" else 1
    row = c["d"] * width + (0 if c["cache"] == "bf16" else 4)                   # one key or value of one head in the cache
    table = 4 * sum(-(-n // c["page"]) for n in lens)
    if c["op"] == "kv":
        rows, fresh = sum(lens) * c["heads"] * 2, sum(new) * c["heads"] * 2
        back = c["batch"] * max(lens) * c["heads"] * 2
        return {"bytes": fresh * (2 * c["d"] + row) + (rows - fresh) * row + back * 2 * c["d"] + table, "flops": 4 * rows * c["d"]}
    pairs = sum(n * t - (n * (n - 1) // 2 if c["causal"] else 0) for n, t in zip(new, lens))
    return {"bytes": 2 * sum(lens) * c["kv_heads"] * row + 4 * sum(new) * c["heads"] * c["d"] + table + 4 * c["heads"] * c["bias"],
            "flops": 4 * pairs * c["heads"] * c["d"]}


def _e4m3_64(x):
    """The nearest e4m3 number, ties to the even mantissa, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "w4":
        n, k = c["n"], c["k"]
        w = torch.empty(n, k, device=s["x"].device, dtype=F64)
        for half in (0, 1):
            bits = (s["codes"].long() >> (4 * half)) & 15
            e, m = (bits >> 1) & 3, (bits & 1).double()
            mag = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1))
            w[:, half::2] = torch.where(bits >= 8, -mag, mag)
        for j in range(s["scales"].shape[1]):
            w[:, j * c["group"]: (j + 1) * c["group"]] *= s["scales"][:, j: j + 1].double()
        out = s["x"].double() @ w.t()
        if c["resid"]:
            out += s["resid"].double()
        return torch.relu(out) if c["relu"] else out
    cu, lens, page, d = s["cu"].tolist(), s["lens"].tolist(), c["page"], c["d"]
    Hk = c["heads"] if c["op"] == "kv" else c["kv_heads"]

    def held(pages, scales, b):
        """Keys or values of sequence b in the order of its positions: [heads, kv_len, d] in 64 bits."""
        ids = s["table"][b, : -(-lens[b] // page)].long()
        rows = []
        for h in range(Hk):
            x = (pages[:, h].contiguous().view(torch.uint8)[ids].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[ids, h]).double()
            if scales is not None:
                x = x * scales[ids, h].double()[..., None]
            rows.append(x.reshape(-1, d)[: lens[b]])
        return torch.stack(rows)

    if c["op"] == "kv":
        back = []
        for pages, scales, x in ((s["k"], s["ks"], s["new_k"]), (s["v"], s["vs"], s["new_v"])):
            out = torch.zeros(c["batch"], max(lens), Hk * d, device=x.device, dtype=F64)
            for b in range(c["batch"]):
                y = x[cu[b]: cu[b + 1]].double().view(-1, Hk, d)
                if c["cache"] != "bf16":
                    most = 127.0 if c["cache"] == "int8" else 448.0
                    unit = (y.abs().amax(-1, keepdim=True) / most).clamp_min(1e-300)
                    y = (torch.round(y / unit) if c["cache"] == "int8" else _e4m3_64(y / unit)) * unit
                first = lens[b] - (cu[b + 1] - cu[b])
                out[b, : lens[b]] = held(pages, scales, b).transpose(0, 1).reshape(lens[b], -1)
                out[b, first: lens[b]] = y.reshape(-1, Hk * d)
            back.append(out)
        return tuple(back)
    H, g = c["heads"], c["heads"] // Hk
    out = torch.zeros(cu[-1], H, d, device=s["q"].device, dtype=F64)
    for b in range(c["batch"]):
        n, t = cu[b + 1] - cu[b], lens[b]
        k, v = held(s["k"], s["ks"], b), held(s["v"], s["vs"], b)
        far = torch.arange(t - n, t, device=k.device)[:, None] - torch.arange(t, device=k.device)[None]
        for h in range(H):
            z = s["q"][cu[b]: cu[b + 1], h * d: (h + 1) * d].double() @ k[h // g].t() * s["scale"]
            if s["bias"] is not None:
                z += s["bias"][h].double()[far.clamp(0, c["bias"] - 1)]
            if c["causal"]:
                z[far < 0] = -math.inf
            out[cu[b]: cu[b + 1], h] = torch.softmax(z, -1) @ v[h // g]
    return out.flatten(1)
