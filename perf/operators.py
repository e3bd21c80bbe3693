"""What is measured of the operators between a layer's q/k/v projections and its output projection: the head norm with the
rotation (`norm_rope`), the paged KV cache as it is written (`write`) and read back (`read`), and the attention of new
tokens over it (`attention`).

Sizes are those of the Qwen3-0.6B / 8B / 32B shaped layers (16 / 32 / 64 query heads over 8 KV heads of 128) and of a GPT-2
shaped layer (12 heads of 64), in bf16 and fp16, with a 16-bit cache or an 8-bit one (e4m3 codes with one power-of-two
exponent for each token and head). A case's `lens` seeds the lengths of its sequences, so that they belong to the case.

Cache pages are [pages, kv_heads, page, head_dim], exponents [pages, kv_heads, page]; a sequence's tokens are found through
its row of the block table. `cu_q` are the offsets of the sequences' new tokens in the packed batch, `kv_len` counts the
cached tokens of a sequence, the new ones among them."""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = {"bf16": 120, "fp16": 8}   # the exponent at which a code over 240 would no longer be finite in the type


def _attention(name, dtype, bits, heads, kv_heads, dim, page, batch, q, past, ragged, lens, decodes=0, causal=True, window=0, lse=False):
    return {"name": name, "op": "attention", "dtype": dtype, "bits": bits, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "batch": batch, "q": q, "past": past, "ragged": ragged, "lens": lens, "decodes": decodes, "causal": causal, "window": window, "lse": lse}


def _norm_rope(name, dtype, heads, kv_heads, dim, tokens, rotary, interleaved, norm, far):
    return {"name": name, "op": "norm_rope", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "tokens": tokens,
            "rotary": rotary, "interleaved": interleaved, "norm": norm, "far": far}


def _cache(op, name, dtype, bits, kv_heads, dim, page, batch, q, past, ragged, lens):
    return {"name": name, "op": op, "dtype": dtype, "bits": bits, "kv_heads": kv_heads, "dim": dim, "page": page, "batch": batch,
            "q": q, "past": past, "ragged": ragged, "lens": lens, "decodes": 0}


def listed():
    return [
        # one user's next token over a short conversation: latency
        _attention("decode_one", "bf16", 16, 16, 8, 128, 16, 1, 1, 700, False, 1),
        # a serving step of a full batch, ragged contexts
        _attention("decode_batch", "bf16", 16, 32, 8, 128, 16, 64, 1, 4095, True, 2),
        # few users with long documents on an 8-bit cache
        _attention("decode_long_8bit", "bf16", 8, 64, 8, 128, 64, 6, 1, 50000, True, 3, lse=True),
        # prefill of a batch of prompts, the heads and lengths of the framework's attention workload
        _attention("prefill", "bf16", 16, 32, 8, 128, 64, 8, 2048, 0, False, 4),
        # one chunk of a long prompt whose beginning is in an 8-bit cache
        _attention("chunk_long_8bit", "bf16", 8, 32, 8, 128, 32, 1, 1000, 16000, False, 5),
        # a continuous batch: some sequences in their prompt, others decoding, heads of 64, a sliding window
        _attention("mixed_window", "fp16", 16, 12, 12, 64, 16, 24, 500, 1500, True, 6, decodes=16, window=1024, lse=True),
        # q and k of a decode step
        _norm_rope("norm_rope_decode", "bf16", 16, 8, 128, 8, 128, False, True, 40000),
        # q and k of a prefill of 8192 tokens in the largest layer
        _norm_rope("norm_rope_prefill", "bf16", 64, 8, 128, 8192, 128, False, True, 131072),
        # a decode step's K and V into the 8-bit cache
        _cache("write", "write_decode_8bit", "bf16", 8, 8, 128, 16, 64, 1, 4095, True, 7),
        # a prefill's K and V into the 8-bit cache
        _cache("write", "write_prefill_8bit", "bf16", 8, 8, 128, 32, 8, 4096, 0, False, 8),
        # a short 16-bit context brought out for an operator that wants plain rows
        _cache("read", "read_short", "fp16", 16, 12, 64, 16, 3, 1, 300, True, 9),
        # long 8-bit contexts brought out whole
        _cache("read", "read_long_8bit", "bf16", 8, 8, 128, 32, 8, 1, 16383, True, 10),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention"] * 6 + ["norm_rope", "norm_rope", "write", "read"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    bits = rng.choice([16, 8])
    dim = rng.choice([128, 128, 64, 96, 80])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    page = rng.choice([16, 16, 32, 64, 128])
    lens = rng.randrange(1 << 30)
    if op == "norm_rope":
        tokens = _log(rng, 1, min(8192, 8192 * 72 // (heads + kv_heads)))
        case = _norm_rope("", rng.choice([dtype, dtype, "fp32"]), heads, kv_heads, dim, tokens, rng.choice([dim, dim, dim // 2]), rng.random() < 0.4,
                          rng.random() < 0.7, _log(rng, 64, 1 << 20))
    elif op in ("write", "read"):
        batch = _log(rng, 1, 128)
        rows = 32000 * 8 * 128 // (kv_heads * dim)
        if op == "write":
            q = rng.choice([1, _log(rng, 1, max(1, min(4096, rows // batch)))])
            past = _log(rng, 1, max(1, 200000 // batch))
        else:
            q, past = 1, _log(rng, 1, max(1, min(16383, 3 * rows // batch)))
        case = _cache(op, "", dtype, bits, kv_heads, dim, page, batch, q, past, True, lens)
    else:
        kind = rng.choice(["decode", "decode", "prefill", "chunk", "mixed", "cross"])
        causal, window, decodes = True, 0, 0
        if kind == "decode":
            batch = _log(rng, 1, 96)
            q = rng.choice([1, 1, 1, 2, 4])
            past = _log(rng, 1, min(60000, 2400000 // (batch * kv_heads)))
            window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
        else:
            # kept within the work of the prefill case: batch * heads * q * keys
            batch = _log(rng, 1, 12)
            room = 8 * 32 * 2048 * 1024 * 128 // (batch * heads * dim)
            if kind == "prefill":
                q, past = _log(rng, 2, max(2, min(4096, int(math.sqrt(room))))), 0
            else:
                q = _log(rng, 2, min(2048, int(math.sqrt(room))))
                past = _log(rng, 1, max(1, min(32000, room // q // 2)))
            if kind == "mixed":
                decodes = batch // 2
            causal = kind != "cross"
            window = rng.choice([0, 0, _log(rng, 16, 2048)]) if causal else 0
        case = _attention("", dtype, bits, heads, kv_heads, dim, page, batch, q, past, True, lens, decodes, causal, window, rng.random() < 0.3)
    del case["name"]
    return case


def _lengths(case):
    """New tokens and cached tokens (the new ones among them, but for cross attention) of each sequence."""
    r = random.Random(case["lens"])
    qs, kvs = [], []
    for b in range(case["batch"]):
        q, past = case["q"], case["past"]
        if case["ragged"]:
            q = q if b == 0 or q <= 4 else r.randint(q // 2, q)
            past = past if b == 0 else r.randint(past // 3, past)
        if b >= case["batch"] - case["decodes"]:
            q = 1
        qs.append(q)
        kvs.append(past if not case.get("causal", True) else past + q)
    return qs, kvs


def _kept(case, q, kv):
    """Pairs of a new token and a cached one that the mask keeps."""
    if not case["causal"]:
        return q * kv
    total = 0
    for i in range(q):
        seen = kv - q + i + 1
        total += min(seen, case["window"]) if case["window"] else seen
    return total


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm_rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * n * size + 4 * case["tokens"], "flops": 10 * n}
    qs, kvs = _lengths(case)
    cell = case["dim"] * case["bits"] // 8 + (1 if case["bits"] == 8 else 0)   # one head's row of the cache
    if case["op"] == "write":
        n = sum(qs) * case["kv_heads"]
        return {"bytes": 2 * n * (case["dim"] * size + cell), "flops": 4 * n * case["dim"]}
    if case["op"] == "read":
        n = sum(kvs) * case["kv_heads"]
        return {"bytes": 2 * n * (case["dim"] * size + cell), "flops": 2 * n * case["dim"]}
    read = 0
    for q, kv in zip(qs, kvs):
        first = max(0, kv - q - case["window"] + 1) if case["window"] else 0
        read += kv - first
    pairs = sum(_kept(case, q, kv) for q, kv in zip(qs, kvs))
    rows = sum(qs) * case["heads"]
    return {"bytes": 2 * rows * case["dim"] * size + 2 * read * case["kv_heads"] * cell + (4 * rows if case["lse"] else 0),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


def _quantise(x, dtype):
    """e4m3 codes and exponents of rows: the least power of two at which the row's largest value is at most 448."""
    x = x.float()
    mant, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(mant == 0, torch.full_like(e, -126), torch.where(mant <= 0.875, e - 9, e - 8).clamp(-126, 120))
    y = torch.ldexp(x, -e[..., None])
    most = torch.where(e >= LARGEST[dtype], 240.0, 448.0)[..., None]
    return torch.minimum(torch.maximum(y, -most), most).to(torch.float8_e4m3fn), e.to(torch.int8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)

    def normal(*shape, dtype=DTYPES[case["dtype"]], scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "norm_rope":
        t, hq, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        qkv = normal(t, (hq + 2 * hk) * d)          # what the fused projection leaves: q, k and v of a token side by side
        s["q"] = qkv[:, :hq * d].view(t, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
        s["q_weight"] = 1 + normal(d, scale=0.2) if case["norm"] else None
        s["k_weight"] = 1 + normal(d, scale=0.2) if case["norm"] else None
        s["positions"] = torch.randint(0, case["far"], (t,), generator=gen, device="cuda", dtype=torch.int32)
        half = case["rotary"] // 2
        s["inv_freq"] = (1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)).float() * (0.25 if case["far"] > 100000 else 1.0)
        s["factor"] = 1.1 if case["far"] > 100000 else 1.0
        s["q_out"] = torch.zeros(t, hq, d, dtype=s["q"].dtype, device="cuda")
        s["k_out"] = torch.zeros(t, hk, d, dtype=s["q"].dtype, device="cuda")
        return s
    qs, kvs = _lengths(case)
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    counts = [-(-kv // page) for kv in kvs]
    pages, width = sum(counts) + 3, max(1, max(counts))
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(qs), width, dtype=torch.int32)
    at = torch.zeros(len(qs), width, dtype=torch.int64)
    taken = 0
    for b, n in enumerate(counts):
        at[b, :n] = torch.arange(taken, taken + n)
        taken += n
    table = order[at.cuda()]
    s["table"] = table.contiguous()
    s["cu_q"] = torch.tensor([sum(qs[:b]) for b in range(len(qs) + 1)], dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(kvs, dtype=torch.int32, device="cuda")
    s["max_q"], s["max_kv"], s["tokens"] = max(qs), max(kvs), sum(qs)
    for name in ("k", "v"):
        rows = normal(pages, hk, page, d, scale=1.0 if name == "k" else 0.7)
        if case["bits"] == 8:
            codes, exps = _quantise(rows, case["dtype"])
            s[name + "_pages"], s[name + "_exp"] = codes, exps
        else:
            s[name + "_pages"], s[name + "_exp"] = rows, None
        del rows
    if case["op"] == "write":
        kv = normal(s["tokens"], 2 * hk * d)
        s["k"] = kv[:, :hk * d].view(-1, hk, d)
        s["v"] = kv[:, hk * d:].view(-1, hk, d)
    elif case["op"] == "read":
        s["cu_kv"] = torch.tensor([sum(kvs[:b]) for b in range(len(kvs) + 1)], dtype=torch.int32, device="cuda")
        s["k_out"] = torch.zeros(sum(kvs), hk, d, dtype=DTYPES[case["dtype"]], device="cuda")
        s["v_out"] = torch.zeros_like(s["k_out"])
    else:
        s["q"] = normal(s["tokens"], case["heads"], d)
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros(s["tokens"], case["heads"], device="cuda") if case["lse"] else None
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------

def _norm(x, weight):
    x = x.float()
    return x if weight is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()


def _rotate(x, cos, sin, rotary, interleaved):
    turned, kept = x[..., :rotary], x[..., rotary:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :rotary // 2], turned[..., rotary // 2:])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, kept), -1)


def _plain_norm_rope(s):
    case = s["case"]
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()
    cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()
    return [_rotate(_norm(x, w), cos, sin, case["rotary"], case["interleaved"]).to(x.dtype)
            for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"]))]


def _owners(s):
    """Sequence and position of each new token."""
    token = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["cu_q"].long(), token, right=True) - 1
    new = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    return b, token - s["cu_q"].long()[b], (s["kv_len"].long() - new)[b] + token - s["cu_q"].long()[b]


def _plain_write(s):
    case = s["case"]
    b, _, position = _owners(s)
    at = (s["table"][b, position // case["page"]].long(), slice(None), position % case["page"])
    if case["bits"] == 8:
        for name in ("k", "v"):
            codes, exps = _quantise(s[name], case["dtype"])
            s[name + "_pages"].view(torch.uint8)[at] = codes.view(torch.uint8)
            s[name + "_exp"][at] = exps
    else:
        s["k_pages"][at], s["v_pages"][at] = s["k"], s["v"]


def _values(s, name):
    pages = s[name + "_pages"].float()
    return pages if s[name + "_exp"] is None else torch.ldexp(pages, s[name + "_exp"][..., None].int())


def _plain_read(s):
    case = s["case"]
    token = torch.arange(s["k_out"].shape[0], device="cuda")
    b = torch.searchsorted(s["cu_kv"].long(), token, right=True) - 1
    position = token - s["cu_kv"].long()[b]
    at = (s["table"][b, position // case["page"]].long(), slice(None), position % case["page"])
    return [_values(s, name)[at].to(DTYPES[case["dtype"]]) for name in ("k", "v")]


def _plain_attention(s):
    case = s["case"]
    hq, hk, d, batch, most = case["heads"], case["kv_heads"], case["dim"], case["batch"], s["max_q"]
    b, i, position = _owners(s)
    q = torch.zeros(batch, most, hq, d, device="cuda")
    q[b, i] = s["q"].float()
    where = torch.zeros(batch, most, dtype=torch.int64, device="cuda")
    where[b, i] = position
    table = s["table"].long()
    keys = table.shape[1] * case["page"]
    k = _values(s, "k")[table].permute(0, 2, 1, 3, 4).reshape(batch, hk, keys, d)
    v = _values(s, "v")[table].permute(0, 2, 1, 3, 4).reshape(batch, hk, keys, d)
    at = torch.arange(keys, device="cuda")
    cached = at[None, :] < s["kv_len"].long()[:, None]
    v = v * cached[:, None, :, None]
    keep = cached[:, None, :].expand(batch, most, keys)
    if case["causal"]:
        keep = keep & (at <= where[..., None])
        if case["window"]:
            keep = keep & (at > where[..., None] - case["window"])
    q = q.view(batch, most, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, -1, d)
    scores = (q @ k.transpose(-1, -2)).view(batch, hk, hq // hk, most, keys).mul_(1 / math.sqrt(d))
    scores.masked_fill_(~keep[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min_(-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(batch, hk, -1, keys) @ v).view(batch, hk, hq // hk, most, d) / total.clamp_min(1e-38)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, hq, d)[b, i].to(s["q"].dtype)
    if s["lse"] is None:
        return [out]
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(batch, most, hq)[b, i]
    return [out, lse]


# ---- the framework's operators ----------------------------------------------------------------------------------------

def _headers(s):
    """The framework's headers (views, cache, batch) of the program's buffers, as it keeps them from step to step."""
    import magnetron_b200 as mb
    case = s["case"]
    kinds = {torch.float32: mb.FLOAT32, torch.float16: mb.FLOAT16, torch.bfloat16: mb.BFLOAT16}

    def tensor(t):
        return None if t is None else mb.Tensor(0, kinds[t.dtype], t.shape, t.stride(), base_ptr=t.data_ptr())

    def pointer(t):
        return None if t is None else t.data_ptr()

    h = {name: tensor(s.get(name)) for name in ("q", "k", "v", "q_weight", "k_weight", "q_out", "k_out", "v_out", "out", "lse")}
    if case["op"] == "norm_rope":
        h["rope"] = mb.Rope(pointer(s["positions"]), pointer(s["inv_freq"]), case["rotary"], interleaved=case["interleaved"], factor=s["factor"])
    else:
        h["cache"] = mb.KVCache(0, kinds[DTYPES[case["dtype"]]], s["k_pages"].shape[0], case["page"], case["kv_heads"], case["dim"], bits=case["bits"],
                                k=pointer(s["k_pages"]), v=pointer(s["v_pages"]), k_exp=pointer(s["k_exp"]), v_exp=pointer(s["v_exp"]))
        h["batch"] = mb.KVBatch(case["batch"], s["table"].shape[1], cu_q=pointer(s["cu_q"]), kv_len=pointer(s["kv_len"]), pages=pointer(s["table"]),
                                max_q=s["max_q"], max_kv=s["max_kv"])
    h["mb"] = mb
    return h


def _own_norm_rope(s, h):
    h["mb"].qk_norm_rope(h["q"], h["k"], h["rope"], h["q_out"], h["k_out"], q_weight=h["q_weight"], k_weight=h["k_weight"], eps=1e-6)
    return [s["q_out"], s["k_out"]]


def _own_write(s, h):
    h["mb"].kv_cache_write(h["cache"], h["batch"], h["k"], h["v"])


def _own_read(s, h):
    h["mb"].kv_cache_read(h["cache"], h["batch"], s["cu_kv"].data_ptr(), h["k_out"], h["v_out"])
    return [s["k_out"], s["v_out"]]


def _own_attention(s, h):
    case = s["case"]
    h["mb"].paged_attention(h["q"], h["cache"], h["batch"], h["out"], lse=h["lse"], causal=case["causal"], window=case["window"])
    return [s["out"]] if s["lse"] is None else [s["out"], s["lse"]]


def run(state):
    op = state["case"]["op"]
    if own:
        if "headers" not in state:
            state["headers"] = _headers(state)
        out = {"norm_rope": _own_norm_rope, "write": _own_write, "read": _own_read, "attention": _own_attention}[op](state, state["headers"])
    else:
        out = {"norm_rope": _plain_norm_rope, "write": _plain_write, "read": _plain_read, "attention": _plain_attention}[op](state)
    # a write's result is the cache itself: codes as the e4m3 values they are, exponents as whole numbers
    return [state[n] for n in ("k_pages", "v_pages", "k_exp", "v_exp") if state[n] is not None] if op == "write" else out


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def _exact_norm_rope(case, s):
    got = []
    half = case["rotary"] // 2
    turn = torch.outer(s["positions"].double(), s["inv_freq"].double())
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.double()
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * w.double()
        z = y.clone()
        for i in range(half):
            m, n = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
            c, t = s["factor"] * turn[:, i, None].cos(), s["factor"] * turn[:, i, None].sin()
            z[..., m] = y[..., m] * c - y[..., n] * t
            z[..., n] = y[..., n] * c + y[..., m] * t
        got.append(z)
    return got


def _exact_codes(x, dtype):
    x = x.double()
    largest = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(largest, -126.0)
    some = largest > 0
    e[some] = torch.ceil(torch.log2(largest[some] / 448)).clamp(-126, 120)
    e = torch.where(largest > 448 * 2.0 ** e, e + 1, e)
    e = torch.where((largest <= 448 * 2.0 ** (e - 1)) & (e > -126) & some, e - 1, e)
    y = x / 2.0 ** e
    most = torch.where(e >= LARGEST[dtype], 240.0, 448.0)
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.minimum(torch.maximum(torch.round(y / step) * step, -most), most), e[..., 0]


def _exact_write(case, s):
    qs, kvs = _lengths(case)
    got = {}
    for name in ("k", "v"):
        pages = s[name + "_pages"].double()
        exps = None if s[name + "_exp"] is None else s[name + "_exp"].clone()
        rows, powers = _exact_codes(s[name], case["dtype"]) if case["bits"] == 8 else (s[name].double(), None)
        table = s["table"].cpu()
        at = 0
        for b, (q, kv) in enumerate(zip(qs, kvs)):
            done = 0
            while done < q:
                position = kv - q + done
                n = min(q - done, case["page"] - position % case["page"])
                p, o = int(table[b, position // case["page"]]), position % case["page"]
                pages[p, :, o:o + n] = rows[at + done:at + done + n].transpose(0, 1)
                if exps is not None:
                    exps[p, :, o:o + n] = powers[at + done:at + done + n].transpose(0, 1).to(torch.int8)
                done += n
            at += q
        got[name] = (pages, exps)
    return [x for x in (got["k"][0], got["v"][0], got["k"][1], got["v"][1]) if x is not None]


def _context(case, s, name, b, kv):
    n = -(-kv // case["page"])
    pages = s["table"][b, :n].long()
    rows = s[name + "_pages"][pages].double()
    if s[name + "_exp"] is not None:
        rows = rows * 2.0 ** s[name + "_exp"][pages].double()[..., None]
    return rows.transpose(0, 1).reshape(case["kv_heads"], n * case["page"], case["dim"])[:, :kv]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        return _exact_norm_rope(case, s)
    if case["op"] == "write":
        return _exact_write(case, s)
    qs, kvs = _lengths(case)
    if case["op"] == "read":
        return [torch.cat([_context(case, s, name, b, kv).transpose(0, 1) for b, kv in enumerate(kvs)]) for name in ("k", "v")]
    out = torch.zeros(s["tokens"], case["heads"], case["dim"], dtype=torch.float64, device="cuda")
    lse = torch.full((s["tokens"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    at = 0
    for b, (q, kv) in enumerate(zip(qs, kvs)):
        k, v = _context(case, s, "k", b, kv), _context(case, s, "v", b, kv)
        col = torch.arange(kv, device="cuda")
        row = kv - q + torch.arange(q, device="cuda")[:, None]
        keep = torch.ones(q, kv, dtype=torch.bool, device="cuda")
        if case["causal"]:
            keep = col <= row
            if case["window"]:
                keep &= row - col < case["window"]
        for h in range(case["heads"]):
            if not kv:
                continue
            z = s["q"][at:at + q, h].double() @ k[h // group].T / math.sqrt(case["dim"])
            z = torch.where(keep, z, torch.full_like(z, -math.inf))
            lse[at:at + q, h] = torch.logsumexp(z, -1)
            out[at:at + q, h] = torch.where(keep, (z - lse[at:at + q, h, None]).exp(), torch.zeros_like(z)) @ v[h // group]
        at += q
    return [out, lse] if case["lse"] else [out]
