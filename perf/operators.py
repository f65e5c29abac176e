"""Speed and exactness cases of the 8-bit linears and the masked attention of ``arbius_amd.ops``.

``run`` computes each operator in its plain form (elementary torch operations in 32 bits), or with
``own`` set through the framework's entry points; ``exact`` computes it from the definition in 64 bits.

* ``linear``: ``ops.linear_int8`` - rows of x quantised to 8 bits with one scale each, times a weight held
  in 8 bits with one scale per output channel: y = act(sx sw (qx . qw) + b + residual).
* ``ln_linear``: ``ops.ln_linear_int8`` - the same product of LayerNorm(x).
* ``attention``: ``ops.masked_attention`` - attention with per-row lengths, documents, causal / prefix
  masks, tanh-capped scores and a bias linear in the distance.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one prompt token through the widest projection of a text-to-image prior: launch latency and the
        # read of the weight
        _linear("linear_one_token", 1, 2048, 8192, act="gelu"),
        # the second feed-forward product of a text tower over 16 padded prompts of 77 tokens
        _linear("linear_text_tower", 1232, 4096, 1024, residual=True),
        # no size a multiple of a tile or of a 16-byte chunk
        _linear("linear_odd_sizes", 1003, 1101, 1333, act="quick_gelu", dtype="fp16"),
        # gated feed-forward of an image UNet's second level (32 x 32 tokens, batch 16)
        _linear("linear_geglu_unet", 16384, 640, 5120, act="geglu"),
        # a wide product over many rows: the matrix cores' rate
        _linear("linear_large", 16384, 8192, 8192),
        # QKV of the prior for one guided task (2 rows of 81 tokens)
        _linear("ln_linear_prior_qkv", 162, 2048, 6144, op="ln_linear"),
        # QKV of an image UNet's first level (64 x 64 tokens, batch 16): memory traffic
        _linear("ln_linear_unet_qkv", 65536, 320, 960, op="ln_linear", bias=False),
        # text tower over a batch of prompts padded to 77 tokens, each with its own length
        _attention("attention_prompts", batch=16, nq=77, nk=77, heads=16, kv_heads=16, dim=64, lengths=True),
        # causal text tower over prompts packed end to end
        _attention("attention_packed_prompts", batch=1, nq=8192, nk=8192, heads=12, kv_heads=12, dim=64, causal=True,
                   doc_tokens=41),
        # long causal prefill with capped scores and shared key / value heads
        _attention("attention_capped_prefill", batch=1, nq=8192, nk=8192, heads=32, kv_heads=8, dim=128, causal=True,
                   softcap=50.0),
        # prefix-causal with a distance bias, odd length, a head width off the tile
        _attention("attention_prefix_bias", batch=2, nq=2047, nk=2047, heads=8, kv_heads=8, dim=80, causal=True,
                   prefix=True, bias=True, dtype="fp16"),
        # one new token for each of four sequences against a long cache, every sequence at its own position
        _attention("attention_one_token", batch=4, nq=1, nk=65537, heads=32, kv_heads=8, dim=128, causal=True,
                   lengths=True, bias=True),
    ]


def _linear(name, m, k, n, op="linear", act="none", bias=True, residual=False, dtype="bf16"):
    case = {"op": op, "m": m, "k": k, "n": n, "act": act, "bias": bias, "residual": residual, "dtype": dtype}
    return dict(case, name=name) if name else case


def _attention(name, batch, nq, nk, heads, kv_heads, dim, causal=False, lengths=False, prefix=False, doc_tokens=0,
               softcap=0.0, bias=False, dtype="bf16"):
    case = {"op": "attention", "batch": batch, "nq": nq, "nk": nk, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "causal": causal, "lengths": lengths, "prefix": prefix, "doc_tokens": doc_tokens, "softcap": softcap,
            "bias": bias, "dtype": dtype}
    return dict(case, name=name) if name else case


def _spread(rng, low, high):
    """An integer of [low, high], even over its logarithm; half of them multiples of 8 where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 8:
        v -= v % 8
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["linear", "linear", "ln_linear", "attention", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "linear":
        m, k, n = _spread(rng, 1, 65536), _spread(rng, 48, 8192), _spread(rng, 48, 8192)
        m = max(1, min(m, 16384 * 8192 * 4096 // (k * n), (1 << 29) // max(k, n)))
        act = rng.choice(["none", "none", "gelu", "quick_gelu", "geglu"])
        return _linear(None, m, k, n + n % 2 if act == "geglu" else n, act=act, bias=rng.random() < 0.7,
                       residual=act == "none" and rng.random() < 0.5, dtype=dtype)
    if op == "ln_linear":
        m, k, n = _spread(rng, 1, 65536), _spread(rng, 48, 2048), _spread(rng, 48, 8192)
        m = max(1, min(m, (1 << 29) // max(k, n)))
        return _linear(None, m, k, n, op=op, act=rng.choice(["none", "gelu", "quick_gelu"]),
                       bias=rng.random() < 0.7, dtype=dtype)
    dim = rng.choice([40, 64, 64, 80, 96, 128, 128, 160, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    form = rng.choice(["prompts", "packed", "prefill", "one_token"])
    bias, softcap = rng.random() < 0.4, rng.choice([0.0, 0.0, 30.0, 50.0])
    if form == "one_token":
        batch, nk = rng.choice([1, 2, 4, 8]), _spread(rng, 64, 65537)
        return _attention(None, batch, rng.choice([1, 1, 1, 2, 5]), nk, heads, kv_heads, dim, causal=True,
                          lengths=True, bias=bias, softcap=softcap, dtype=dtype)
    if form == "prompts":
        n = _spread(rng, 1, 300)
        return _attention(None, rng.choice([1, 3, 16, 32]), n, n, heads, kv_heads, dim, lengths=True,
                          causal=rng.random() < 0.3, bias=bias, softcap=softcap, dtype=dtype)
    n = _spread(rng, 200, 8192)
    if form == "packed":
        return _attention(None, 1, n, n, heads, kv_heads, dim, causal=rng.random() < 0.5,
                          doc_tokens=_spread(rng, 5, 1000), bias=bias, softcap=softcap, dtype=dtype)
    n = min(n, 4096)
    return _attention(None, rng.choice([1, 2]), n, n, heads, kv_heads, dim, causal=True, prefix=rng.random() < 0.5,
                      bias=bias, softcap=softcap, dtype=dtype)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    st = dict(case)
    if case["op"] != "attention":
        m, k, n = case["m"], case["k"], case["n"]
        # activations as a transformer has them: a few channels far wider than the rest
        wide = 1.0 + 15.0 * (torch.rand(k, generator=gen, device="cuda") < 0.01).float()
        st["x"] = (normal(m, k) * wide).to(dtype)
        w = normal(n, k) / math.sqrt(k)
        ws = w.abs().amax(dim=1) / 127.0
        # the weight in 8 bits as a program keeps it: rows laid out on 16-byte boundaries
        rows = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device="cuda")
        rows[:, :k] = torch.round(w / ws[:, None]).clamp(-127, 127).to(torch.int8)
        st["wq"], st["ws"] = rows[:, :k], ws
        st["b"] = normal(n).to(dtype) if case["bias"] else None
        st["residual"] = normal(m, n).to(dtype) if case["residual"] else None
        if case["op"] == "ln_linear":
            st["gamma"], st["beta"] = (1.0 + 0.1 * normal(k)).to(dtype), (0.1 * normal(k)).to(dtype)
        return st
    B, nq, nk, H = case["batch"], case["nq"], case["nk"], case["heads"]
    st["q"] = normal(B, nq, H, case["dim"]).to(dtype)
    st["k"] = normal(B, nk, case["kv_heads"], case["dim"]).to(dtype)
    st["v"] = normal(B, nk, case["kv_heads"], case["dim"]).to(dtype)
    for name in ("lengths", "prefixes", "documents", "start", "slopes"):
        st[name] = None
    if case["lengths"]:
        low = max(nq, nk // 2) if nq < nk else 0
        st["lengths"] = torch.randint(low, nk + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    if nq < nk:                     # new tokens at the end of each sequence's cache
        st["start"] = st["lengths"] - nq
    if case["prefix"]:
        st["prefixes"] = torch.randint(0, nk // 2 + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    if case["doc_tokens"]:
        count = max(1, nk // case["doc_tokens"])
        share = torch.rand(count, generator=gen, device="cuda", dtype=torch.float64) + 0.2
        ends = torch.round(share.cumsum(0) * (nk / share.sum())).to(torch.int32)
        st["documents"] = torch.cat([torch.zeros_like(ends[:1]), ends]).contiguous()
    if case["bias"]:
        st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    if own:
        return _own(st)
    return _plain_attention(st) if st["op"] == "attention" else _plain_linear(st)


def _own(st):
    from arbius_amd import ops
    if st["op"] == "attention":
        return ops.masked_attention(st["q"], st["k"], st["v"], causal=st["causal"], lengths=st["lengths"],
                                    prefix=st["prefixes"], documents=st["documents"], q_start=st["start"],
                                    softcap=st["softcap"] or None, slopes=st["slopes"])
    w = ops.Int8Rows(st["wq"], st["ws"])
    act = None if st["act"] == "none" else st["act"]
    if st["op"] == "ln_linear":
        return ops.ln_linear_int8(st["x"], st["gamma"], st["beta"], 1e-5, w, st["b"], act=act)
    return ops.linear_int8(st["x"], w, st["b"], residual=st["residual"], act=act)


def _gelu(x):
    return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))


def _plain_linear(st):
    x = st["x"].float()
    if st["op"] == "ln_linear":
        x = x - x.mean(dim=1, keepdim=True)
        x = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + 1e-5)
        x = x * st["gamma"].float() + st["beta"].float()
    top = x.abs().amax(dim=1, keepdim=True)
    # next to a half step 32 bits do not say which side a value is on
    q = torch.round(x.double() * 127.0 / top.double()).nan_to_num(0.0).float()
    y = (q @ st["wq"].float().t()) * (top / 127.0) * st["ws"]
    if st["b"] is not None:
        y = y + st["b"].float()
    if st["residual"] is not None:
        y = y + st["residual"].float()
    if st["act"] == "gelu":
        y = _gelu(y)
    elif st["act"] == "quick_gelu":
        y = y * torch.sigmoid(1.702 * y)
    elif st["act"] == "geglu":
        half = y.shape[1] // 2
        y = y[:, :half] * _gelu(y[:, half:])
    return y.to(st["x"].dtype)


def _allowed(st, dev):
    """[batch, nq, nk]: which keys each query sees."""
    B, nq, nk = st["batch"], st["nq"], st["nk"]
    j = torch.arange(nk, device=dev)[None, None, :]
    p = torch.arange(nq, device=dev)[None, :, None].expand(B, nq, 1)
    if st["start"] is not None:
        p = p + st["start"].long()[:, None, None]
    ok = torch.ones(B, nq, nk, dtype=torch.bool, device=dev)
    if st["causal"]:
        ahead = j <= p
        if st["prefixes"] is not None:
            ahead = ahead | (j < st["prefixes"].long()[:, None, None])
        ok = ok & ahead
    if st["lengths"] is not None:
        ok = ok & (j < st["lengths"].long()[:, None, None])
    if st["documents"] is not None:
        off = st["documents"].long()
        dp = torch.bucketize(p.contiguous(), off, right=True)
        dj = torch.bucketize(j.contiguous(), off, right=True)
        ok = ok & (dp == dj) & (p < off[-1]) & (p >= off[0])
    return ok, p, j


def _plain_attention(st):
    group = st["heads"] // st["kv_heads"]
    q = st["q"].float().transpose(1, 2).contiguous()
    k = st["k"].float().permute(0, 2, 3, 1).repeat_interleave(group, dim=1).contiguous()
    v = st["v"].float().transpose(1, 2).repeat_interleave(group, dim=1).contiguous()
    s = torch.matmul(q, k) * (1.0 / math.sqrt(st["dim"]))
    if st["softcap"]:
        s = torch.tanh(s / st["softcap"]) * st["softcap"]
    ok, p, j = _allowed(st, s.device)
    if st["slopes"] is not None:
        s = s - st["slopes"][None, :, None, None] * (p - j).abs().float()[:, None]
    s = s.masked_fill(~ok[:, None], float("-inf"))
    s = torch.exp(s - s.amax(dim=-1, keepdim=True).clamp_min(-1e30))
    total = s.sum(dim=-1, keepdim=True)
    o = torch.matmul(s, v) / torch.where(total > 0, total, torch.ones_like(total))
    return o.transpose(1, 2).to(st["q"].dtype).contiguous()


# ------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] != "attention":
        return _exact_linear(st)
    B, nq, nk, H = case["batch"], case["nq"], case["nk"], case["heads"]
    group = H // case["kv_heads"]
    out = torch.zeros(B, nq, H, case["dim"], dtype=torch.float64, device="cuda")
    at = torch.arange(nk, device="cuda")
    for b in range(B):
        first = int(st["start"][b]) if st["start"] is not None else 0
        own_at = torch.arange(first, first + nq, device="cuda")
        # every mask is a run [low, high) of keys
        low, high = torch.zeros_like(own_at), torch.full_like(own_at, nk)
        if case["causal"]:
            shown = int(st["prefixes"][b]) if case["prefix"] else 0
            high = torch.clamp(own_at + 1, min=shown, max=nk)
        if case["doc_tokens"]:
            off = st["documents"].long()
            doc = (off[None, :] <= own_at[:, None]).sum(dim=1) - 1
            inside = (doc >= 0) & (doc < off.numel() - 1)
            doc = doc.clamp(0, off.numel() - 2)
            low = torch.maximum(low, off[doc])
            high = torch.where(inside, torch.minimum(high, off[doc + 1]), low)
        if case["lengths"]:
            high = torch.clamp(high, max=int(st["lengths"][b]))
        seen = (at[None, :] >= low[:, None]) & (at[None, :] < high[:, None])
        some = high > low
        for h in range(H):
            q, k, v = st["q"][b, :, h].double(), st["k"][b, :, h // group].double(), st["v"][b, :, h // group].double()
            s = (q @ k.t().contiguous()) / math.sqrt(case["dim"])
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            if st["slopes"] is not None:
                s = s - st["slopes"][h].double() * (own_at[:, None] - at[None, :]).abs().double()
            s = torch.softmax(torch.where(seen, s, torch.full_like(s, -math.inf))[some], dim=1)
            out[b, some, h] = s @ v
    return out


def _exact_linear(st):
    x = st["x"].double()
    if st["op"] == "ln_linear":
        mean = x.mean(dim=1, keepdim=True)
        var = x.var(dim=1, unbiased=False, keepdim=True)
        x = (x - mean) / torch.sqrt(var + 1e-5) * st["gamma"].double() + st["beta"].double()
    largest = x.abs().max(dim=1, keepdim=True).values
    q = torch.where(largest > 0, torch.round(x * 127.0 / largest), torch.zeros_like(x))
    y = torch.matmul(q, st["wq"].double().t().contiguous()) * (largest / 127.0) * st["ws"].double()[None, :]
    for term in (st["b"], st["residual"]):
        if term is not None:
            y = y + term.double()
    if st["act"] == "quick_gelu":
        return y / (1.0 + torch.exp(-1.702 * y))
    gate = y[:, y.shape[1] // 2:] if st["act"] == "geglu" else y
    phi = 0.5 * torch.special.erfc(-gate / math.sqrt(2.0))
    if st["act"] == "geglu":
        return y[:, :y.shape[1] // 2] * gate * phi
    return y * phi if st["act"] == "gelu" else y


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] != "attention":
        m, k, n = case["m"], case["k"], case["n"]
        out = n // 2 if case["act"] == "geglu" else n
        size = 2 * m * k + n * k + 4 * n + 2 * m * out + (2 * n if case["bias"] else 0)
        size += (2 * m * n if case["residual"] else 0) + (4 * k if case["op"] == "ln_linear" else 0)
        return {"bytes": size, "flops": 2.0 * m * n * k}
    B, nq, nk, H, D = case["batch"], case["nq"], case["nk"], case["heads"], case["dim"]
    # keys a query sees, on average over the random lengths, prefixes and documents
    if case["doc_tokens"]:
        count = max(1, nk // case["doc_tokens"])
        keys, read = (nk / count) * (0.55 if case["causal"] else 1.1), nk
    elif case["lengths"]:
        read = 0.75 * nk if nq < nk else 0.5 * nk
        keys = read * (0.5 if case["causal"] and nq == nk else 1.0)
    elif case["causal"]:
        keys, read = nk * (0.5 + (1.0 / 24 if case["prefix"] else 0.0)), nk
    else:
        keys, read = nk, nk
    size = 2 * B * (2 * nq * H * D + 2 * read * case["kv_heads"] * D)
    return {"bytes": size, "flops": 4.0 * B * H * nq * max(1.0, keys) * D}
