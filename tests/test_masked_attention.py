"""``ops.masked_attention`` against its definition in 64 bits (masks built key by key), on the CPU reference and on
the HIP kernels.

Tolerance.  With w the exact softmax weights, V = sum_j w_j |v_j|: the weights enter the second product
rounded to the input type (half a step each, u = finfo.eps / 2), scores are fp32 sums of exact products and are
off by less than 2^-13 here (|scale q.k| < 64, cap tanh within cap 2^-21), which moves a weight by 2^-12 of
itself at most; the output is rounded once: |o - ref| <= (u + 2^-12) V + u |ref| (+ 2^-25 in fp16's subnormals)."""
import math

import pytest
import torch

from arbius_amd import ops
from arbius_amd.models import layers
from arbius_amd.models.clip_text import CLIPTextConfig, CLIPTextEncoder
from arbius_amd.models.xlmr import MCLIPText, XLMRConfig

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def i32(v):
    return torch.tensor(v, dtype=torch.int32)


def seen_keys(b, i, nk, o):
    """The keys query i of batch row b sees, from the masks' definitions."""
    start = o.get("q_start", 0)
    p = (int(start[b]) if isinstance(start, torch.Tensor) else start) + i
    docs, prefix, lengths = o.get("documents"), o.get("prefix"), o.get("lengths")
    ok = torch.ones(nk, dtype=torch.bool)
    j = torch.arange(nk)
    first, shown = 0, None
    if docs is not None:
        off = (docs[b] if docs.dim() == 2 else docs).tolist()
        t = [t for t in range(len(off) - 1) if off[t] <= p < off[t + 1]]
        if not t:
            return ~ok, p
        first = off[t[0]]
        ok &= (j >= first) & (j < off[t[0] + 1])
        if prefix is not None:
            shown = int((prefix[b] if prefix.dim() == 2 else prefix)[t[0]])
    elif prefix is not None:
        shown = int(prefix[b])
    if o.get("causal"):
        ok &= (j <= p) | ((j < first + shown) if shown is not None else torch.zeros_like(ok))
    if lengths is not None:
        ok &= j < int(lengths[b])
    return ok, p


def definition(q, k, v, o):
    B, Nq, H, D = q.shape
    Nk, group = k.shape[1], H // k.shape[2]
    scale = o.get("scale") or 1.0 / math.sqrt(D)
    out, mag = torch.zeros(B, Nq, H, D, dtype=torch.float64), torch.zeros(B, Nq, H, D, dtype=torch.float64)
    j = torch.arange(Nk)
    for b in range(B):
        runs = [seen_keys(b, i, Nk, o) for i in range(Nq)]
        ok = torch.stack([r[0] for r in runs])
        p = torch.tensor([r[1] for r in runs])
        some = ok.any(dim=1)
        for h in range(H):
            kk = k[b, :, h // group].double()
            vv = v[b, :, h // group].double()
            s = (q[b, :, h].double() @ kk.t()) * scale
            if o.get("softcap"):
                s = o["softcap"] * torch.tanh(s / o["softcap"])
            if o.get("slopes") is not None:
                s = s - o["slopes"][h].double() * (p[:, None] - j).abs()
            s = torch.where(ok, s, torch.full_like(s, -math.inf))[some]
            w = torch.softmax(s, dim=1)
            used = ok.any(dim=0)                      # values no query sees stay out
            out[b, some, h] = w[:, used] @ vv[used]
            mag[b, some, h] = w[:, used] @ vv[used].abs()
    return out, mag


def check(y, want, mag):
    u = torch.finfo(y.dtype).eps / 2
    y = y.cpu().double()
    assert not bool(y.isnan().any())
    over = (y - want).abs() - ((u + 2.0 ** -12) * mag + u * want.abs() + 2.0 ** -25)
    assert bool((over <= 0).all()), f"over the bound by {over.max().item():.3g}"


def to(device, o):
    return {n: t.to(device) if isinstance(t, torch.Tensor) else t for n, t in o.items()}


def run(q, k, v, o, device):
    return ops.masked_attention(q.to(device), k.to(device), v.to(device), **to(device, o))


def slopes(H):
    return 2.0 ** (-8.0 * torch.arange(1, H + 1, dtype=torch.float32) / H)


def spread(n, step):
    """n offsets, 0 .. step * n, documents of every length from 0 to 3 among them."""
    return i32([0] + sorted(min(step * n, j * 3 // 2) for j in range(n - 1)) + [step * n])


CASES = {
    "plain": dict(shape=(2, 77, 77, 3, 3, 64)),
    "one": dict(shape=(1, 1, 1, 1, 1, 8)),
    "one key": dict(shape=(2, 70, 1, 2, 2, 32)),
    "one query": dict(shape=(3, 1, 200, 4, 2, 64), q_start=199, causal=True),
    "wide head": dict(shape=(1, 40, 70, 2, 1, 256), causal=True),
    "head 40": dict(shape=(2, 33, 65, 4, 4, 40)),
    "head 80": dict(shape=(1, 129, 129, 2, 2, 80), causal=True),
    "head 96": dict(shape=(1, 64, 64, 2, 2, 96), softcap=5.0),
    "head 160": dict(shape=(1, 100, 100, 2, 1, 160), causal=True, slopes=slopes(2)),
    "head 200": dict(shape=(1, 50, 131, 2, 2, 200)),
    "groups": dict(shape=(2, 61, 61, 8, 2, 64), causal=True),
    "groups of 3": dict(shape=(1, 90, 90, 6, 2, 32), causal=True, slopes=slopes(6), softcap=20.0),
    "multi-query": dict(shape=(2, 5, 300, 16, 1, 128), causal=True, q_start=295),
    "lengths": dict(shape=(6, 77, 77, 2, 2, 64), lengths=i32([0, 1, 5, 63, 64, 77])),
    "lengths past the end": dict(shape=(3, 20, 20, 2, 2, 64), lengths=i32([-5, 1000, 2 ** 31 - 1])),
    "causal lengths": dict(shape=(3, 150, 150, 2, 2, 64), causal=True, lengths=i32([10, 0, 150])),
    "prefix": dict(shape=(4, 140, 140, 2, 2, 64), causal=True, prefix=i32([0, 1, 70, 140])),
    "prefix past the end": dict(shape=(2, 30, 30, 2, 2, 64), causal=True, prefix=i32([-3, 2 ** 31 - 1])),
    "documents": dict(shape=(1, 300, 300, 2, 2, 64), documents=i32([0, 5, 64, 64, 65, 200, 300])),
    "documents causal": dict(shape=(1, 300, 300, 2, 2, 64), causal=True, documents=i32([0, 5, 64, 65, 200, 300])),
    "documents with gaps": dict(shape=(1, 200, 200, 2, 2, 64), documents=i32([7, 30, 130])),
    "documents past the end": dict(shape=(1, 100, 100, 2, 2, 64), documents=i32([0, 60, 400])),
    "documents per row": dict(shape=(2, 90, 90, 2, 2, 64), documents=i32([[0, 40, 90], [10, 20, 70]])),
    "documents prefix": dict(shape=(1, 160, 160, 2, 2, 64), causal=True, documents=i32([0, 50, 120, 160]),
                             prefix=i32([10, 0, 1000])),
    "documents prefix per row": dict(shape=(2, 80, 80, 2, 2, 64), causal=True, documents=i32([0, 50, 80]),
                                     prefix=i32([[10, 0], [3, 9]])),
    "documents lengths": dict(shape=(2, 90, 90, 2, 2, 64), documents=i32([0, 40, 90]), lengths=i32([60, 20])),
    "one document": dict(shape=(1, 70, 70, 1, 1, 64), documents=i32([0, 70])),
    "softcap": dict(shape=(2, 100, 100, 2, 2, 64), causal=True, softcap=2.0),
    "softcap 50 far over it": dict(shape=(1, 80, 80, 2, 2, 64), softcap=50.0, scale=3.0),
    "slopes": dict(shape=(2, 130, 130, 4, 4, 64), slopes=slopes(4)),
    "rising slopes": dict(shape=(1, 66, 66, 2, 2, 64), causal=True, slopes=torch.tensor([-0.05, 0.0])),
    "starts": dict(shape=(4, 3, 257, 4, 2, 64), causal=True, q_start=i32([0, 100, 254, 300]), slopes=slopes(4)),
    "starts before the first key": dict(shape=(2, 4, 40, 2, 2, 64), causal=True, q_start=i32([-2, -100])),
    "start past every key": dict(shape=(1, 4, 40, 2, 2, 64), causal=True, q_start=2 ** 31 - 5),
    "cached rows": dict(shape=(4, 2, 700, 8, 2, 128), causal=True, q_start=i32([10, 400, 0, 698]),
                        lengths=i32([12, 402, 2, 700])),
    "long cache, few rows": dict(shape=(1, 1, 5003, 4, 2, 64), causal=True, q_start=5002, slopes=slopes(4)),
    "long cache, short lengths": dict(shape=(2, 1, 5000, 4, 2, 64), lengths=i32([0, 130]), softcap=30.0),
    # 8 waves, two on the keys
    "two waves on the keys": dict(shape=(1, 200, 700, 2, 1, 64), causal=True, q_start=500),
    "two waves, head 96, bias": dict(shape=(1, 130, 640, 2, 2, 96), slopes=slopes(2), lengths=i32([601])),
    "two waves, head 128, cap": dict(shape=(2, 97, 1100, 1, 1, 128), causal=True, q_start=i32([1000, 3]),
                                     softcap=30.0),
    "two waves, head 24, all": dict(shape=(1, 550, 550, 3, 1, 24), causal=True, softcap=10.0, slopes=slopes(3),
                                    documents=i32([0, 40, 520, 550]), prefix=i32([9, 0, 40])),
    # key ranges: few of them, more than 64, one that sees nothing
    "ranges of a few rows": dict(shape=(2, 7, 2000, 4, 2, 64), causal=True, q_start=i32([1993, 300])),
    "more than 64 ranges": dict(shape=(1, 1, 12000, 2, 2, 32), lengths=i32([11990]), slopes=slopes(2) / 64),
    "ranges, wide head": dict(shape=(1, 2, 3000, 2, 1, 256), causal=True, q_start=2998, softcap=20.0),
    "ranges, nothing seen": dict(shape=(3, 1, 3000, 2, 2, 128), lengths=i32([0, -1, 129])),
    # document searches: empty ones in a row, more than one step of 64 and of 64 x 64 offsets
    "empty documents in a row": dict(shape=(1, 200, 200, 1, 1, 32), documents=i32([0] + [60] * 150 + [61, 130] +
                                                                                  [131] * 70 + [200])),
    "documents of one or two": dict(shape=(1, 1400, 1400, 1, 1, 8), documents=spread(1100, 2)),
    "thousands of documents": dict(shape=(1, 90, 130, 1, 1, 16), q_start=20, causal=True,
                                   documents=i32([min(j // 60, 130) for j in range(9000)])),
    # positions far from the keys, where fp32 holds neither them nor the distances
    "slopes from far behind": dict(shape=(2, 3, 400, 2, 2, 64), q_start=i32([2 ** 30 + 1, 77777777]),
                                   slopes=slopes(2) / 8, lengths=i32([400, 130])),
    "slopes from far ahead": dict(shape=(1, 40, 200, 2, 2, 64), q_start=i32([-2 ** 30]), slopes=slopes(2)),
    "falling and rising far": dict(shape=(1, 1, 5000, 2, 2, 64), q_start=2 ** 31 - 9,
                                   slopes=torch.tensor([2.0 ** -4, -2.0 ** -5])),
    "smallest cap and largest": dict(shape=(1, 50, 90, 2, 2, 64), softcap=2.0 ** -10),
    "negative scale": dict(shape=(1, 40, 300, 2, 2, 64), scale=-0.2, causal=True, softcap=2.0 ** 10),
    "all": dict(shape=(2, 190, 190, 6, 3, 80), causal=True, documents=i32([3, 90, 180]), prefix=i32([20, 5]),
                lengths=i32([190, 100]), softcap=10.0, slopes=slopes(6), scale=0.2),
}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", CASES)
def test_against_the_definition(device, dtype, name):
    o = dict(CASES[name])
    B, Nq, Nk, H, Hkv, D = o.pop("shape")
    dt = DTYPES[dtype]
    q, k, v = randn(B, Nq, H, D, seed=1, dtype=dt), randn(B, Nk, Hkv, D, seed=2, dtype=dt), \
        randn(B, Nk, Hkv, D, seed=3, dtype=dt)
    y = run(q, k, v, o, device)
    assert y.dtype == dt and tuple(y.shape) == (B, Nq, H, D)
    check(y, *definition(q, k, v, o))


POISONED = {
    "lengths": dict(shape=(3, 70, 200, 2, 2, 64), lengths=i32([0, 64, 131])),
    "documents": dict(shape=(1, 210, 210, 2, 1, 64), documents=i32([0, 50, 130, 150])),
    "cache": dict(shape=(3, 1, 4000, 4, 2, 128), causal=True, q_start=i32([0, 77, 3000]), lengths=i32([1, 78, 2001])),
    "causal": dict(shape=(1, 100, 300, 2, 2, 80), causal=True),
    "two waves on the keys": dict(shape=(1, 150, 800, 1, 1, 128), lengths=i32([707])),
    "head 160": dict(shape=(1, 40, 200, 1, 1, 160), documents=i32([0, 30, 100])),
    "head 256": dict(shape=(1, 3, 900, 1, 1, 256), causal=True, q_start=500),
}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", ["nan", "inf", "lowest"])
@pytest.mark.parametrize("name", POISONED)
def test_masked_places_may_hold_anything(device, dtype, bad, name):
    o = dict(POISONED[name])
    B, Nq, Nk, H, Hkv, D = o.pop("shape")
    dt = DTYPES[dtype]
    val = {"nan": float("nan"), "inf": float("inf"), "lowest": torch.finfo(dt).min}[bad]
    q, k, v = randn(B, Nq, H, D, seed=1, dtype=dt), randn(B, Nk, Hkv, D, seed=2, dtype=dt), \
        randn(B, Nk, Hkv, D, seed=3, dtype=dt)
    clean = run(q, k, v, o, device)
    for b in range(B):
        unseen = ~torch.stack([seen_keys(b, i, Nk, o)[0] for i in range(Nq)]).any(dim=0)
        k[b, unseen], v[b, unseen] = val, val
    y = run(q, k, v, o, device)
    assert not bool(y.isnan().any()) and torch.equal(y, clean)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("val", [float("nan"), float("inf"), -float("inf")])
def test_a_value_reaches_only_the_queries_that_see_it(device, val):
    """V row 50 of a causal row set, V row 20 of one document: queries before it / of the others stay clean."""
    q, k, v = (randn(1, 140, 2, 64, seed=s, dtype=torch.bfloat16) for s in (1, 2, 3))
    at_i = torch.arange(140)
    for o, at, hit in ((dict(causal=True), 50, at_i >= 50),
                       (dict(documents=i32([0, 10, 30, 140])), 20, (at_i >= 10) & (at_i < 30))):
        clean = run(q, k, v, o, device).cpu()
        w = v.clone()
        w[0, at, 0, 5] = val
        y = run(q, k, w, o, device).cpu()
        rest = torch.ones_like(clean, dtype=torch.bool)
        rest[0, hit, 0, 5] = False
        assert torch.equal(y[rest], clean[rest])
        got = y[0, hit, 0, 5]
        assert bool(got.isnan().all()) if math.isnan(val) else bool((got == val).all())


# values that are seen at a weight too small for 32 bits: parts of a split cache, the two-wave plan, one run of tiles
SEEN = {
    "split cache": dict(shape=(1, 1, 6000, 1, 1, 64), slopes=torch.tensor([0.5])),
    "split cache, heads": dict(shape=(2, 2, 5000, 4, 2, 128), causal=True, q_start=4000,
                               slopes=torch.tensor([0.5, 1.0, 2.0, 0.25])),
    "two waves on the keys": dict(shape=(1, 700, 700, 1, 1, 64), slopes=torch.tensor([2.0])),
    "one wave, late maximum": dict(shape=(1, 40, 400, 8, 1, 80), causal=True, q_start=360,
                                   slopes=torch.full((8,), 2.0)),
    "head 256": dict(shape=(1, 3, 900, 1, 1, 256), q_start=890, slopes=torch.tensor([1.0])),
}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", SEEN)
def test_a_seen_value_shows_at_any_weight(device, dtype, name):
    """NaN and infinities that a query sees far away, where a distance bias leaves a weight of 0 in 32 bits: NaN, the
    infinity, or NaN of both signs, in those channels and no others, however the keys are divided."""
    o = dict(SEEN[name])
    B, Nq, Nk, H, Hkv, D = o.pop("shape")
    dt = DTYPES[dtype]
    q, k, v = randn(B, Nq, H, D, seed=1, dtype=dt), randn(B, Nk, Hkv, D, seed=2, dtype=dt), \
        randn(B, Nk, Hkv, D, seed=3, dtype=dt)
    clean = run(q, k, v, o, device).cpu()
    inf, at = float("inf"), 10 if o.get("q_start") else Nk - 5
    v[0, at, 0, 5], v[0, at, 0, 9], v[0, at, 0, 12] = float("nan"), inf, -inf
    v[0, at, 0, 14], v[0, Nk // 2 - 40, 0, 14] = inf, -inf
    y = run(q, k, v, o, device).cpu()
    hit, G = y[0, :, :H // Hkv], H // Hkv
    assert bool(hit[..., 5].isnan().all()) and bool(hit[..., 14].isnan().all())
    assert bool((hit[..., 9] == inf).all()) and bool((hit[..., 12] == -inf).all())
    for d in (5, 9, 12, 14):
        y[0, :, :G, d] = clean[0, :, :G, d]
    assert torch.equal(y, clean)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nk,heads,start",
                         [(140, 140, 2, 0), (1, 6000, 2, 5990), (700, 700, 1, 0), (2, 300, 4, 290)])
def test_scores_that_are_all_minus_infinity(device, dtype, nq, nk, heads, start):
    """Keys, but none with a score above -inf: 0 / 0, where no keys give zeros; one finite score is enough for a row."""
    dt = DTYPES[dtype]
    q, k, v = (randn(3, n, heads, 64, seed=s, dtype=dt) for n, s in ((nq, 1), (nk, 2), (nk, 3)))
    q[..., 0], k[1, :, :, 0] = 1.0, -float("inf")
    k[2, 1:, :, 0] = -float("inf")
    o = dict(causal=True, q_start=start, lengths=i32([0, nk, nk]))
    y = run(q, k, v, o, device).cpu()
    assert not bool(y[0].any()) and bool(y[1].isnan().all())
    # (batch row 2: the one key weighs 1)
    assert torch.equal(y[2], v[2, :1].expand(nq, -1, -1))


@pytest.mark.parametrize("device", DEVICES)
def test_many_small_weights_next_to_a_large_one(device):
    """One key of weight 1 and 4000 of 2^-20 each: the small ones keep their bits, also in fp16."""
    for dt in DTYPES.values():
        q, k, v = torch.zeros(1, 1, 1, 32), torch.zeros(1, 4001, 1, 32), torch.zeros(1, 4001, 1, 32)
        q[..., 0], k[:, 1:, :, 0], v[:, 1:, :, 0] = 1.0, -13.8125, 1000.0
        v[:, 0, :, 1] = 1.0
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
        check(run(q, k, v, dict(scale=1.0), device), *definition(q, k, v, dict(scale=1.0)))


@pytest.mark.parametrize("device", DEVICES)
def test_a_nan_key_or_query_stays_with_its_rows(device):
    q, k, v = (randn(1, 80, 2, 64, seed=s, dtype=torch.bfloat16) for s in (1, 2, 3))
    clean = run(q, k, v, dict(causal=True), device).cpu()
    k2, q2 = k.clone(), q.clone()
    k2[0, 70, 1], q2[0, 33, 0, 3] = float("nan"), float("nan")
    y = run(q2, k2, v, dict(causal=True), device).cpu()
    assert bool(y[0, 70:, 1].isnan().all()) and bool(y[0, 33, 0].isnan().all())
    y[0, 70:, 1], y[0, 33, 0] = clean[0, 70:, 1], clean[0, 33, 0]
    assert torch.equal(y, clean)


@pytest.mark.parametrize("device", DEVICES)
def test_strided_views(device):
    qkv = randn(2, 90, 3, 4, 64, seed=5, dtype=torch.bfloat16).to(device)
    o = dict(causal=True, lengths=i32([90, 31]))
    y = ops.masked_attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], **to(device, o))
    assert torch.equal(y, ops.masked_attention(*(qkv[:, :, i].contiguous() for i in range(3)), **to(device, o)))
    # head-major caches, and one key / value set shared by every batch row
    kh, vh = (randn(2, 2, 90, 64, seed=s, dtype=torch.bfloat16).to(device).transpose(1, 2) for s in (6, 7))
    y = ops.masked_attention(qkv[:, :, 0], kh, vh, **to(device, o))
    assert torch.equal(y, ops.masked_attention(qkv[:, :, 0].contiguous(), kh.contiguous(), vh.contiguous(),
                                               **to(device, o)))
    ke, ve = kh[:1].expand(2, -1, -1, -1), vh[:1].expand(2, -1, -1, -1)
    y = ops.masked_attention(qkv[:, :, 0], ke, ve, causal=True)
    assert torch.equal(y, ops.masked_attention(qkv[:, :, 0], ke.contiguous(), ve.contiguous(), causal=True))
    # index tensors that are columns or rows of others
    both = i32([[90, 1], [31, 2]]).to(device)
    with pytest.raises(ValueError):
        ops.masked_attention(qkv[:, :, 0], kh, vh, lengths=both[:, 0])
    docs = i32([[0, 40, 90, 7], [5, 6, 60, 7]]).to(device)[:, :3]
    y = ops.masked_attention(qkv[:, :, 0], kh, vh, documents=docs)
    assert torch.equal(y, ops.masked_attention(qkv[:, :, 0], kh, vh, documents=docs.contiguous()))


@pytest.mark.parametrize("device", DEVICES)
def test_token_strides_of_any_size(device):
    """Keys 8 MiB apart, a single key whose token stride is that or nothing, keys that are all the same memory."""
    q = randn(1, 3, 2, 64, seed=1, dtype=torch.bfloat16).to(device)
    far = torch.zeros(2 * (1 << 22) + 256, dtype=torch.bfloat16, device=device)
    for n, stride in ((3, 1 << 22), (1, 1 << 23), (1, 0), (5, 0), (9, 8)):
        k = far.as_strided((1, n, 2, 64), (128, stride, 64, 1))
        v = far.as_strided((1, n, 2, 64), (128, stride, 64, 1), 64)
        far[:1 << 14] = randn(1 << 14, seed=n).to(far)
        far[(1 << 23):] = randn(256, seed=n + 1).to(far)
        got, o = ops.masked_attention(q, k, v), dict(causal=False)
        check(got, *definition(q.cpu(), k.cpu().clone(), v.cpu().clone(), o))


@pytest.mark.parametrize("device", DEVICES)
def test_strides_of_single_sizes(device):
    """One batch row, one token, one head: their strides are never used, so any will do; index tensors of one element
    cut out of others too."""
    store = randn(1 << 13, seed=1, dtype=torch.bfloat16).to(device)
    for b, nq, nk, h, hkv in ((1, 3, 5, 2, 2), (2, 1, 1, 2, 2), (2, 3, 5, 1, 1), (1, 1, 1, 1, 1)):
        def odd(n, heads, at):
            full = (512, 64 * heads, 64)
            strides = [st if size > 1 else st + 3 for size, st in zip((b, n, heads), full)]
            return store.as_strided((b, n, heads, 64), (*strides, 1), at)
        q, k, v = odd(nq, h, 0), odd(nk, hkv, 2048), odd(nk, hkv, 4096)
        got = ops.masked_attention(q, k, v, causal=True)
        dense = (t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
        assert torch.equal(got, ops.masked_attention(*dense, causal=True))
    pair = i32([[2, 7], [1, 7]]).to(device)
    got = ops.masked_attention(*(t[:1] for t in (q, k, v)), causal=True, lengths=pair[1:, 0], q_start=pair[:1, 0],
                               prefix=pair[:1, 0])
    assert torch.equal(got, ops.masked_attention(*(t[:1] for t in (q, k, v))))


@pytest.mark.parametrize("device", DEVICES)
def test_scale_of_zero(device):
    q, k, v = (randn(2, 40, 2, 64, seed=s, dtype=torch.float16) for s in (1, 2, 3))
    for o in (dict(scale=0.0, causal=True), dict(scale=0.0, softcap=3.0, lengths=i32([40, 7]))):
        got = run(q, k, v, o, device)
        check(got, *definition(q, k, v, dict(o, scale=1e-30)))


@pytest.mark.parametrize("device", DEVICES)
def test_batch_rows_do_not_touch_each_other(device):
    q, k, v = (randn(8, 100, 4, 64, seed=s, dtype=torch.bfloat16).to(device) for s in (1, 2, 3))
    n = i32([100, 3, 77, 64, 65, 1, 50, 99]).to(device)
    y = ops.masked_attention(q, k, v, lengths=n, causal=True, slopes=slopes(4).to(device))
    with ops.plan_batch(1):
        group = ops.masked_attention(q, k, v, lengths=n, causal=True, slopes=slopes(4).to(device))
        for b in range(8):
            one = ops.masked_attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], lengths=n[b:b + 1], causal=True,
                                       slopes=slopes(4).to(device))
            assert torch.equal(one[0], group[b])
    assert torch.equal(y, ops.masked_attention(q, k, v, lengths=n, causal=True, slopes=slopes(4).to(device)))


@pytest.mark.parametrize("device", DEVICES)
def test_empty_shapes(device):
    q, k = torch.ones(2, 3, 4, 64, dtype=torch.bfloat16, device=device), \
        torch.ones(2, 0, 2, 64, dtype=torch.bfloat16, device=device)
    assert not bool(ops.masked_attention(q, k, k).any())
    assert tuple(ops.masked_attention(q[:, :0], k, k).shape) == (2, 0, 4, 64)
    assert tuple(ops.masked_attention(q[:0], k[:0], k[:0]).shape) == (0, 3, 4, 64)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    q, k = torch.ones(2, 3, 4, 64, dtype=torch.bfloat16, device=device), \
        torch.ones(2, 5, 2, 64, dtype=torch.bfloat16, device=device)
    n, att = i32([1, 2]).to(device), ops.masked_attention
    for bad in (lambda: att(q[0], k, k), lambda: att(q, k, k[:, :4]), lambda: att(q[:1], k, k),
                lambda: att(q[..., :32], k, k), lambda: att(q[:, :, :3], k, k),
                lambda: att(q, k, k, scale=float("nan")), lambda: att(q, k, k, softcap=0.0),
                lambda: att(q, k, k, softcap=-1.0), lambda: att(q, k, k, softcap=float("inf")),
                lambda: att(q, k, k, softcap=1e4), lambda: att(q, k, k, softcap=1e-4), lambda: att(q, k, k, scale=1e7),
                lambda: att(q[:1].expand(2 ** 31, -1, -1, -1), *2 * (k[:1].expand(2 ** 31, -1, -1, -1),)),
                lambda: att(q, k, k, q_start=-1), lambda: att(q, k, k, q_start=2 ** 31),
                lambda: att(q, k, k, lengths=n[:1]), lambda: att(q, k, k, q_start=n[:1]),
                lambda: att(q, k, k, documents=n[:1]), lambda: att(q, k, k, documents=n[:0]),
                lambda: att(q, k, k, documents=n[0]), lambda: att(q, k, k, prefix=n),
                lambda: att(q, k, k, causal=True, prefix=n[:1]),
                lambda: att(q, k, k, causal=True, documents=n, prefix=n),
                lambda: att(q, k, k, slopes=slopes(2).to(device)), lambda: att(q, k, k, slopes=0.5),
                lambda: att(q, k, k, slopes=slopes(4).double().to(device))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: att(q, k.half(), k), lambda: att(q, k, k, lengths=n.long()),
                lambda: att(q, k, k, lengths=[1, 2]), lambda: att(q, k, k, causal=True, prefix=n.float())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="inference only"):
        att(q.clone().requires_grad_(), k, k)


@pytest.mark.parametrize("device", DEVICES)
def test_no_operand_asks_for_a_gradient(device):
    q, s = torch.ones(1, 3, 4, 64, dtype=torch.bfloat16, device=device), slopes(4).to(device).requires_grad_()
    with pytest.raises(RuntimeError, match="inference only"):
        ops.masked_attention(q, q, q, slopes=s)
    with torch.no_grad():
        assert torch.equal(ops.masked_attention(q, q, q, slopes=s), ops.masked_attention(q, q, q, slopes=s.detach()))
    rows = ops.quantize_rows(q[0, 0])
    with pytest.raises(RuntimeError, match="inference only"):
        ops.Int8Rows(rows.q, rows.scale.clone().requires_grad_())


@pytest.mark.gpu
def test_gpu_refusals(cuda):
    q = torch.ones(1, 3, 2, 72, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(TypeError):
        ops.masked_attention(q.float(), q.float(), q.float())
    for t in (q[..., :4], q[..., 4:], torch.ones(1, 3, 2, 264, dtype=torch.bfloat16, device=cuda)):
        with pytest.raises(ValueError):
            ops.masked_attention(t, t, t)
    with pytest.raises(ValueError):
        ops.masked_attention(q[..., :64].transpose(1, 3), q, q)
    with pytest.raises(TypeError):
        ops.masked_attention(q, q, q, lengths=i32([3]))


@pytest.mark.gpu
def test_cache_past_32_bit_offsets(cuda):
    """A cache whose last keys lie more than 2^32 bytes behind its first."""
    n, row = 70000, 32768
    store = torch.empty(n, row, dtype=torch.bfloat16, device=cuda)
    k, v = store[None, :, :128].view(1, n, 2, 64), store[None, :, 4096:4224].view(1, n, 2, 64)
    gen = torch.Generator(device=cuda).manual_seed(1)
    for t in (store[:, :128], store[:, 4096:4224]):
        t.copy_(torch.randn(n, 128, generator=gen, device=cuda))
    q = torch.randn(1, 2, 4, 64, generator=gen, device=cuda).to(torch.bfloat16)
    o = dict(causal=True, q_start=n - 2, slopes=torch.tensor([0.0, 2.0 ** -12, 0.5, 0.0]))
    y = run(q, k, v, o, cuda)
    assert torch.equal(y, run(q, k.contiguous(), v.contiguous(), o, cuda))
    check(y, *definition(q.cpu(), k.cpu(), v.cpu(), o))


@pytest.mark.gpu
def test_many_batch_rows(cuda):
    B = 70000
    q, k, v = (randn(64, n, 1, 32, seed=s, dtype=torch.bfloat16).to(cuda).repeat(-(-B // 64), 1, 1, 1)[:B]
               for s, n in ((1, 2), (2, 5), (3, 5)))
    y = ops.masked_attention(q, k, v, lengths=torch.full((B,), 4, dtype=torch.int32, device=cuda))
    check(y[:64], *definition(q[:64].cpu(), k[:64].cpu(), v[:64].cpu(), dict(lengths=i32([4] * 64))))
    assert torch.equal(y, y[:64].repeat(-(-B // 64), 1, 1, 1)[:B])


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nk", [(100, 100), (1, 6000)])
def test_streams_and_graph_replays(cuda, nq, nk):
    """Two graphs over caches that grow between replays; lengths and positions are read on the device."""
    q = [randn(2, nq, 4, 64, seed=s, dtype=torch.bfloat16).to(cuda) for s in (1, 2)]
    k, v = (randn(2, nk, 2, 64, seed=s, dtype=torch.bfloat16).to(cuda) for s in (3, 4))
    n, start = i32([nk, 1]).to(cuda), i32([0, 0]).to(cuda)
    o = dict(causal=True, lengths=n, q_start=start, softcap=20.0)
    want = ops.masked_attention(q[0], k, v, **o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.masked_attention(q[0], k, v, **o)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.masked_attention(q[i], k, v, **o)
        graphs.append((g, y))
    for step in range(1, 5):
        n.copy_(i32([nk // step, step * nk // 5]))
        start.copy_(i32([max(0, nk // step - nq), step]))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(graphs[i][1], ops.masked_attention(q[i], k, v, **o))


@pytest.mark.gpu
def test_calls_at_once_on_two_streams(cuda):
    """Split attention and 8-bit linears in flight together: each call has its own workspace."""
    q, k, v = (randn(2, n, h, 64, seed=s, dtype=torch.bfloat16).to(cuda) for s, n, h in ((1, 1, 4), (2, 6000, 2),
                                                                                         (3, 6000, 2)))
    x, w = (randn(n, 640, seed=n, dtype=torch.bfloat16).to(cuda) for n in (700, 640))
    w = ops.quantize_rows(w)
    starts = [dict(causal=True, q_start=n) for n in (5999, 3000)]
    want = [ops.masked_attention(q, k, v, **o) for o in starts] + [ops.linear_int8(x, w), ops.linear_int8(x[:3], w)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for step in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append((ops.masked_attention(q, k, v, **starts[i]), ops.linear_int8(x[:3] if i else x, w)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, y in got[i]:
            assert torch.equal(a, want[i]) and torch.equal(y, want[2 + i])


# ------------------------------------------------------------------ as the text towers use it
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("int8", [False, True])
def test_packed_prompts_through_the_text_towers(device, int8):
    """Prompts packed end to end give what each gives alone: a run of 8-bit linears and masked attention."""
    dt = torch.bfloat16 if device == "cuda" else torch.float32
    lens = [5, 30, 1, 77, 12]
    off = i32([0] + list(torch.tensor(lens).cumsum(0)))
    ids = torch.randint(3, 900, (sum(lens),), generator=torch.Generator().manual_seed(1))
    clip = layers.init_weights(CLIPTextEncoder(CLIPTextConfig(vocab=1000, width=128, layers=2, heads=2, mlp=256)), 1)
    xlmr = layers.init_weights(MCLIPText(XLMRConfig(vocab=1000, width=128, layers=2, heads=2, mlp=256, max_pos=100,
                                                    proj_dim=64)), 2)
    for model in (clip, xlmr):
        model.to(device=device, dtype=dt).eval()
        ids[off[1:].long() - 1] = 999                       # every prompt ends with its EOS
        if int8:
            assert layers.int8_linears(model) == (8 if model is clip else 9)
        full, pooled = model.forward_packed(ids.to(device), off.to(device))
        for t, n in enumerate(lens):
            row = ids[int(off[t]):int(off[t + 1])][None].to(device)
            one, pool = model(row) if model is clip else model(row, n)
            part = full[int(off[t]):int(off[t + 1])]
            # bf16: two layers of roundings at 2^-8 each, an 8-bit step where one flips; fp32: sums in another order
            tol = 2e-4 if dt == torch.float32 and not int8 else 0.03
            assert (part.float() - one[0].float()).norm() <= tol * one[0].float().norm()
            assert (pooled[t].float() - pool[0].float()).norm() <= tol * pool[0].float().norm()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("int8", [False, True])
def test_prompts_that_do_not_fit_are_marked(device, int8):
    """Empty prompts, prompts longer than the position table, tokens before and behind all prompts, offsets past the
    tokens: NaN for those, the others' features untouched, and no index leaves its table."""
    dt = torch.bfloat16 if device == "cuda" else torch.float32
    off = i32([4, 30, 30, 150, 160, 171, 400]).to(device)               # 26 tokens, none, 120, 10, 11, too many
    ids = torch.randint(3, 900, (200,), generator=torch.Generator().manual_seed(1)).to(device)
    clip = layers.init_weights(CLIPTextEncoder(CLIPTextConfig(vocab=1000, width=128, layers=2, heads=2, mlp=256)), 1)
    xlmr = layers.init_weights(MCLIPText(XLMRConfig(vocab=1000, width=128, layers=2, heads=2, mlp=256, max_pos=100,
                                                    proj_dim=64)), 2)
    good = torch.tensor([True, False, False, True, True, False])
    for model in (clip, xlmr):
        model.to(device=device, dtype=dt).eval()
        if int8:
            layers.int8_linears(model)
        full, pooled = model.forward_packed(ids, off)
        assert torch.equal(pooled.isnan().all(dim=1).cpu(), ~good) and bool(pooled[good].isfinite().all())
        assert bool(full[:4].isnan().all()) and bool(full[4:30].isfinite().all())
        fit = i32([0, 26, 36, 47]).to(device)
        alone = model.forward_packed(torch.cat([ids[4:30], ids[150:171]]), fit)[1]
        # the same prompts at other places of other key tiles: two layers of roundings, an 8-bit step where one flips
        assert (pooled[good].float() - alone.float()).norm() <= (2e-4 if device == "cpu" and not int8 else 0.03) * \
            alone.float().norm()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("int8", [False, True])
def test_prompts_without_any_token(device, int8):
    dt = torch.bfloat16 if device == "cuda" else torch.float32
    clip = layers.init_weights(CLIPTextEncoder(CLIPTextConfig(vocab=1000, width=128, layers=2, heads=2, mlp=256)), 1)
    xlmr = layers.init_weights(MCLIPText(XLMRConfig(vocab=1000, width=128, layers=2, heads=2, mlp=256, max_pos=100,
                                                    proj_dim=64)), 2)
    none = torch.zeros(0, dtype=torch.long, device=device)
    for model, width in ((clip, 128), (xlmr, 64)):
        model.to(device=device, dtype=dt).eval()
        if int8:
            layers.int8_linears(model)
        for off in ([0, 0, 0], [0, 5], [0]):
            full, pooled = model.forward_packed(none, i32(off).to(device))
            assert tuple(full.shape) == (0, 128) and full.dtype == pooled.dtype == dt
            assert tuple(pooled.shape) == (len(off) - 1, width) and bool(pooled.isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
def test_packed_prompts_in_a_graph(cuda, int8):
    """One graph over ids and offsets that change between replays, with eager work in between: other prompts, empty
    ones, one too long, and the same again."""
    from arbius_amd.models.graphs import GraphedCall
    clip = layers.init_weights(CLIPTextEncoder(CLIPTextConfig(vocab=1000, width=128, layers=2, heads=2, mlp=256)), 1)
    xlmr = layers.init_weights(MCLIPText(XLMRConfig(vocab=1000, width=128, layers=2, heads=2, mlp=256, max_pos=100,
                                                    proj_dim=64)), 2)
    packs = [[0, 30, 60, 130, 200], [0, 0, 77, 77, 90], [0, 1, 2, 3, 200], [5, 40, 41, 99, 150], [0, 30, 60, 130, 200]]
    for model in (clip, xlmr):
        model.to(device=cuda, dtype=torch.bfloat16).eval()
        if int8:
            layers.int8_linears(model)
        ids = [torch.randint(3, 900, (200,), generator=torch.Generator().manual_seed(s)).to(cuda)
               for s in (1, 2, 3, 4, 1)]
        with torch.no_grad():
            want = [tuple(t.clone() for t in model.forward_packed(i, i32(off).to(cuda))) for i, off in zip(ids, packs)]
            graph = GraphedCall(model.forward_packed, [ids[0], i32(packs[0]).to(cuda)])
            for _ in range(2):
                for i, off, (full, pooled) in zip(ids, packs, want):
                    got = graph(i, i32(off).to(cuda))
                    torch.cuda.synchronize()
                    assert torch.equal(got[0].nan_to_num(7.0), full.nan_to_num(7.0))
                    assert torch.equal(got[1].nan_to_num(7.0), pooled.nan_to_num(7.0))
                    model.forward_packed(i, i32(off).to(cuda))
