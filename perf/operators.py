"""What is measured of the attention operators with a learned relative position bias.

Query i and key j of a sequence with sq queries and sk keys are r = j - (i + sk - sq) positions apart (bottom-right
aligned). A table of shape (num_buckets, heads) holds one learned number per bucket of r and head:

    S = scale * Q K^T + table[bucket(r), head],   P = softmax(S),   O = P V

  op "prompt"  attention over whole prompts, the forward pass alone
  op "train"   the forward pass, then dQ, dK, dV and the table's gradient for a given dO
  op "decode"  one or a few new tokens of every sequence against a cache of keys and values, lengths per sequence
  op "bias"    the bias itself, (heads, sq, sk), and the table's gradient for a given gradient of it

Buckets: with n = |r|, half of the table for r <= 0 and half for r > 0 (bidirectional), or the whole table for
n = max(-r, 0). A side of nb buckets gives the distances below e = nb // 2 a bucket each; bucket e + t takes those with
log(n / e) / log(max_distance / e) * (nb - e) >= t in real numbers, and the last bucket everything beyond.
"""

import math
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a short prompt of one user: the call's latency
        dict(name="prompt_short", op="prompt", dtype="bf16", batch=1, packed=0, lens=1, sq=128, sk=128, hq=8, hkv=8, d=64, causal=1, buckets=32, far=128),
        # prompts of different lengths packed into one batch, grouped heads, as a server collects them
        dict(name="prompt_packed_gqa", op="prompt", dtype="bf16", batch=12, packed=1, lens=7, sq=2048, sk=2048, hq=32, hkv=8, d=128, causal=1, buckets=32, far=128),
        # one long prompt behind an earlier part of it (more keys than queries), odd lengths
        dict(name="prompt_chunk", op="prompt", dtype="fp16", batch=1, packed=0, lens=1, sq=1777, sk=6001, hq=16, hkv=2, d=128, causal=1, buckets=64, far=1024),
        # training step of a decoder layer, grouped heads: the largest case
        dict(name="train_causal_gqa", op="train", dtype="bf16", batch=2, packed=0, lens=1, sq=4096, sk=4096, hq=16, hkv=4, d=128, causal=1, buckets=32, far=128),
        # training step of an encoder layer, both directions
        dict(name="train_encoder", op="train", dtype="fp16", batch=8, packed=0, lens=1, sq=512, sk=512, hq=12, hkv=12, d=64, causal=0, buckets=32, far=128),
        # training on packed documents of odd lengths
        dict(name="train_packed", op="train", dtype="bf16", batch=9, packed=1, lens=3, sq=1531, sk=1531, hq=8, hkv=4, d=64, causal=1, buckets=32, far=256),
        # float32, as gradient checks and small models use it
        dict(name="train_fp32", op="train", dtype="fp32", batch=2, packed=0, lens=1, sq=200, sk=200, hq=4, hkv=4, d=64, causal=0, buckets=32, far=128),
        # one new token of one sequence: the smallest step of generation
        dict(name="decode_one", op="decode", dtype="bf16", batch=1, lens=5, sq=1, sk=1025, hq=32, hkv=8, d=128, buckets=32, far=128),
        # one new token of many sequences with long caches
        dict(name="decode_batch", op="decode", dtype="bf16", batch=48, lens=11, sq=1, sk=8192, hq=32, hkv=8, d=128, buckets=32, far=128),
        # a few drafted tokens at once
        dict(name="decode_draft", op="decode", dtype="fp16", batch=6, lens=2, sq=5, sk=4001, hq=16, hkv=4, d=64, buckets=32, far=512),
        # the bias of an encoder layer as a tensor, and its gradient
        dict(name="bias_encoder", op="bias", dtype="fp16", sq=512, sk=512, hq=12, two=1, buckets=32, far=128),
        # the same for long sequences, odd sizes
        dict(name="bias_long", op="bias", dtype="bf16", sq=4095, sk=4099, hq=16, two=0, buckets=32, far=128),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["prompt", "train", "train", "decode", "decode", "bias"])
    side = rng.choice([8, 16, 32, 64])
    far = _log_int(rng, side, 2048)
    if op == "bias":
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), sq=_log_int(rng, 1, 4095), sk=_log_int(rng, 17, 4099),
                    hq=rng.choice([1, 4, 6, 8, 12, 16]), two=rng.choice([0, 1]), buckets=side, far=far)
    hkv, group, d = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4]), rng.choice([64, 128])
    if op == "decode":
        return dict(op=op, dtype=rng.choice(["bf16", "fp16"]), batch=_log_int(rng, 1, 48), lens=rng.randrange(1000), sq=rng.choice([1, 1, 1, 2, 3, 8]),
                    sk=_log_int(rng, 33, 8192), hq=hkv * group, hkv=hkv, d=d, buckets=side, far=far)
    dtype = rng.choice(["bf16", "fp16"])
    small = op == "train" and rng.random() < 0.15
    if small:
        dtype = "fp32"
    sk = _log_int(rng, 17, 256 if small else 4096)
    packed = rng.choice([0, 1])
    causal = rng.choice([0, 1])
    sq = sk if packed or rng.random() < 0.6 else max(1, min(sk, _log_int(rng, 1, sk)))
    hq = hkv * group
    most = (1 + causal) * 16 * 4096 * 4096  # cells of score matrices that cost no more than the largest listed case
    if hq * sk * sk > most:
        hq, hkv = group, 1
    room = most // (max(hq, side) * sk * sk)
    batch = _log_int(rng, 1, max(1, min(2 if small else 16, room)))
    return dict(op=op, dtype=dtype, batch=batch, packed=packed, lens=rng.randrange(1000), sq=sq, sk=sk, hq=hq, hkv=hkv, d=d, causal=causal, buckets=side, far=far)


def _two_sided(case):
    if case["op"] == "bias":
        return bool(case["two"])
    return case["op"] != "decode" and not case["causal"]


def _lengths(case):
    """Keys per sequence. Packed batches and caches hold sequences of different lengths, the longest as long as the case says."""
    if case["op"] != "decode" and not case["packed"]:
        return [case["sk"]] * case["batch"]
    rng = random.Random(case["lens"])
    return [case["sk"]] + [max(1, round(case["sk"] * rng.uniform(0.1, 1.0))) for _ in range(case["batch"] - 1)]


def _starts(case):
    """First distance of the buckets 1, 2, ... of a side, by whole numbers."""
    nb = case["buckets"] // (2 if _two_sided(case) else 1)
    e = nb // 2
    m = nb - e
    starts = list(range(1, e))
    for t in range(m):
        n = max(e, int(e * (case["far"] / e) ** (t / m)) - 2)
        while n ** m * e ** t < case["far"] ** t * e ** m:
            n += 1
        starts.append(n)
    return starts


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(t)  # noqa: E731
    s = dict(case=case, table=rn(case["buckets"], case["hq"]))
    if case["op"] == "bias":
        s["grad"] = rn(case["hq"], case["sq"], case["sk"])
        s["table"].requires_grad_()
        return s
    lens, d = _lengths(case), case["d"]
    if case["op"] == "decode":
        s["q"] = rn(case["batch"], case["sq"], case["hq"], d)
        s["k"], s["v"] = rn(case["batch"], case["sk"], case["hkv"], d), rn(case["batch"], case["sk"], case["hkv"], d)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return s
    if case["packed"]:
        total = sum(lens)
        s["q"], s["k"], s["v"] = rn(total, case["hq"], d), rn(total, case["hkv"], d), rn(total, case["hkv"], d)
        ends = [0]
        for n in lens:
            ends.append(ends[-1] + n)
        s["cu"], s["max"] = torch.tensor(ends, dtype=torch.int32, device="cuda"), max(lens)
    else:
        s["q"] = rn(case["batch"], case["sq"], case["hq"], d)
        s["k"], s["v"] = rn(case["batch"], case["sk"], case["hkv"], d), rn(case["batch"], case["sk"], case["hkv"], d)
    if case["op"] == "train":
        s["dout"] = rn(*s["q"].shape)
        for n in ("q", "k", "v", "table"):
            s[n].requires_grad_()
    return s


# ---------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------
def _buckets(r, case):
    starts = torch.tensor(_starts(case), device=r.device)
    if _two_sided(case):
        return torch.bucketize(r.abs(), starts, right=True) + (r > 0) * (case["buckets"] // 2)
    return torch.bucketize((-r).clamp(min=0), starts, right=True)


def _scores(q, k, table, len_q, len_k, case, causal):
    """q (b, hq, sq, d), k (b, hq, sk, d) in float32; len_q, len_k (b or 1, 1, 1): S. What is not visible gets -inf."""
    i = torch.arange(q.shape[2], device=q.device)[None, :, None]
    j = torch.arange(k.shape[2], device=q.device)[None, None, :]
    r = j - (i + len_k - len_q)
    seen = (i < len_q) & (j < len_k) & ((r <= 0) if causal else True)
    s = torch.matmul(q, k.transpose(-1, -2)) * case["d"] ** -0.5
    s += table.t()[:, _buckets(r, case)].transpose(0, 1)
    return s.masked_fill_(~seen[:, None], -math.inf)


def _by_bucket(x, shift, case):
    """x (b, h, sq, sk) summed over the pairs of each bucket, where query i and key j are j - i - shift apart (shift: b or 1): (b, h, buckets)."""
    sq, sk = x.shape[2:]
    # the sums along the diagonals: rows from the last to the first, each a place further right, over one another
    x = torch.nn.functional.pad(x.flip(2), (0, sq)).flatten(2)[..., : sq * (sk + sq - 1)].unflatten(2, (sq, sk + sq - 1))
    along = x.sum(2, dtype=torch.float64)  # column c: j - i = c - (sq - 1)
    b = _buckets(torch.arange(sk + sq - 1, device=x.device) - (sq - 1) - shift.view(-1, 1), case)
    which = (b[..., None] == torch.arange(case["buckets"], device=x.device)).double()
    return torch.matmul(along, which)


def _softmax(s):
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m.masked_fill(m == -math.inf, 0.0))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_attention(s, case):
    t, group = TYPES[case["dtype"]], case["hq"] // case["hkv"]
    wide = lambda x: x.float().transpose(1, 2)  # noqa: E731
    q, k, v, table, dout = s["q"], s["k"], s["v"], s["table"].float(), s.get("dout")
    if case.get("packed"):  # sequences side by side, the short ones filled up
        cu = s["cu"].long()
        n = cu[1:] - cu[:-1]
        at = torch.arange(s["max"], device=q.device)[None, :]
        rows = (cu[:-1, None] + at).clamp(max=q.shape[0] - 1)
        back = at < n[:, None]
        q, k, v = q[rows], k[rows], v[rows]
        dout = None if dout is None else dout[rows] * back[:, :, None, None]
        len_q = len_k = n[:, None, None]
    elif case["op"] == "decode":
        len_q, len_k = torch.tensor(case["sq"], device=q.device).view(1, 1, 1), s["lens"].long()[:, None, None]
    else:
        len_q, len_k = (torch.tensor(case[x], device=q.device).view(1, 1, 1) for x in ("sq", "sk"))
    q, k, v = wide(q), wide(k).repeat_interleave(group, 1), wide(v).repeat_interleave(group, 1)
    scores = _scores(q, k, table, len_q, len_k, case, case["op"] == "decode" or case["causal"])
    p = _softmax(scores)
    del scores
    lay = lambda x: (x.transpose(1, 2)[back] if case.get("packed") else x.transpose(1, 2)).to(t)  # noqa: E731
    o = torch.matmul(p, v)
    if case["op"] != "train":
        return lay(o)
    do = wide(dout)
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds -= (do * o).sum(-1, keepdim=True)
    ds *= p
    del p
    dq = torch.matmul(ds, k) * case["d"] ** -0.5
    dk = torch.matmul(ds.transpose(-1, -2), q) * case["d"] ** -0.5
    shared = lambda x: x.unflatten(1, (case["hkv"], group)).sum(2)  # noqa: E731
    dtable = _by_bucket(ds, len_k - len_q, case).sum(0)  # (hq, buckets)
    return [lay(o), lay(dq), lay(shared(dk)), lay(shared(dv)), dtable.t().to(t)]


def _plain_bias(s, case):
    t, grad = TYPES[case["dtype"]], s["grad"]
    h, sq, sk = grad.shape
    i, j = torch.arange(sq, device=grad.device)[:, None], torch.arange(sk, device=grad.device)[None, :]
    bias = s["table"].float().t()[:, _buckets(j - (i + sk - sq), case)].to(t)
    dtable = _by_bucket(grad.float()[None], torch.tensor(sk - sq, device=grad.device), case)[0]
    return [bias, dtable.t().to(t)]


def _own(s, case):
    if "flashback-cute_b200" not in sys.path:
        sys.path.insert(0, "flashback-cute_b200")
    import flashback_cute as fb

    if case["op"] == "bias":
        bias = fb.flashback_relpos_bias(s["table"], case["sq"], case["sk"], max_distance=case["far"], bidirectional=bool(case["two"]))
        return [bias.detach(), torch.autograd.grad(bias, s["table"], s["grad"])[0]]
    if case["op"] == "decode":
        return fb.flashback_attn_relpos_decode(s["q"], s["k"], s["v"], s["lens"], s["table"], max_distance=case["far"])
    if case["packed"]:
        out = fb.flashback_attn_relpos_varlen_func(s["q"], s["k"], s["v"], s["table"], s["cu"], s["cu"], s["max"], s["max"],
                                                   max_distance=case["far"], causal=bool(case["causal"]))
    else:
        out = fb.flashback_attn_relpos_func(s["q"], s["k"], s["v"], s["table"], max_distance=case["far"], causal=bool(case["causal"]))
    if case["op"] == "prompt":
        return out
    return [out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["table"]), s["dout"])]


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    with torch.no_grad():
        return _plain_bias(state, case) if case["op"] == "bias" else _plain_attention(state, case)


def _pairs(case):
    """Visible (query, key) pairs of one head, over all sequences."""
    n = 0
    for sk in _lengths(case):
        sq = sk if case.get("packed") else case["sq"]
        if case["op"] == "decode" or case["causal"]:
            hidden = min(sq, sk) * (min(sq, sk) - 1) // 2 + max(0, sq - sk) * sk  # keys behind their query
            n += sq * sk - hidden
        else:
            n += sq * sk
    return n


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    table = case["buckets"] * case["hq"]
    if case["op"] == "bias":
        cells = case["hq"] * case["sq"] * case["sk"]
        return {"bytes": size * (2 * cells + 2 * table), "flops": cells}
    lens, d = _lengths(case), case["d"]
    rows_k = sum(lens)
    rows_q = rows_k if case.get("packed") else case["batch"] * case["sq"]
    q, k = rows_q * case["hq"] * d, rows_k * case["hkv"] * d
    product = 2 * _pairs(case) * case["hq"] * d
    if case["op"] == "train":  # q, k, v, dO in; O and dQ, dK, dV out
        return {"bytes": size * (4 * q + 4 * k + 2 * table), "flops": 7 * product}
    return {"bytes": size * (2 * q + 2 * k + table), "flops": 2 * product}


# ---------------------------------------------------------------------------------------------------
# the definition in 64 bits: one (sequence, head) at a time, the derivative taken through the formula
# ---------------------------------------------------------------------------------------------------
def _bucket_of(n, nb, far):
    """Bucket of distance n on a side of nb buckets."""
    e = nb // 2
    if n < e:
        return n
    t = 0
    while t + 1 < nb - e and n ** (nb - e) * e ** (t + 1) >= far ** (t + 1) * e ** (nb - e):
        t += 1
    return e + t


def _bucket_row(lo, hi, case):
    """Buckets of the positions lo, lo + 1, ..., hi apart."""
    two = _two_sided(case)
    nb = case["buckets"] // (2 if two else 1)
    memo = {}

    def side(n):
        n = min(n, case["far"])
        if n not in memo:
            memo[n] = _bucket_of(n, nb, case["far"])
        return memo[n]

    return torch.tensor([(side(-r) if r <= 0 else (nb + side(r) if two else 0)) for r in range(lo, hi + 1)], device="cuda")


def exact(case, seed):
    s = prepare(case, seed)
    table = s["table"].detach().double()
    if case["op"] == "bias":
        sq, sk = case["sq"], case["sk"]
        row = _bucket_row(1 - sk, sq - 1 + max(0, sk - sq), case)  # r runs from -(sk - 1) to sq - 1
        at = row[(torch.arange(sk, device="cuda")[None, :] - torch.arange(sq, device="cuda")[:, None] - (sk - sq)) + sk - 1]
        bias, dtable = torch.empty_like(s["grad"], dtype=torch.float64), torch.zeros_like(table)
        for h in range(case["hq"]):
            bias[h] = table[:, h][at]
            for t in range(case["buckets"]):
                dtable[t, h] = s["grad"][h].double()[at == t].sum()
        return [bias, dtable]
    train, group, scale = case["op"] == "train", case["hq"] // case["hkv"], case["d"] ** -0.5
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    out = torch.empty_like(q)
    if train:
        do = s["dout"].double()
        dq, dk, dv, dtable = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(table)
    at = 0
    for b, n in enumerate(_lengths(case)):
        if case.get("packed"):
            rq = rk = slice(at, at + n)
            at += n
            part = lambda x, rows, h: x[rows, h]  # noqa: E731
        else:
            rq, rk = (b, slice(None)), (b, slice(0, n))
            part = lambda x, rows, h: x[rows[0], rows[1], h]  # noqa: E731
        sq = n if case.get("packed") else case["sq"]
        r = torch.arange(n, device="cuda")[None, :] - torch.arange(sq, device="cuda")[:, None] - (n - sq)
        low = min(0, 1 - n)
        row = _bucket_row(low, max(sq - 1, n - 1), case)
        which = row[r - low]
        hidden = (r > 0) if case["op"] == "decode" or case["causal"] else torch.zeros_like(r, dtype=torch.bool)
        for h in range(case["hq"]):
            qh, kh, vh = part(q, rq, h), part(k, rk, h // group), part(v, rk, h // group)
            x = qh @ kh.T
            x.mul_(scale).add_(table[:, h][which])
            x[hidden] = -math.inf
            lse = torch.logsumexp(x, -1, keepdim=True)
            p = torch.exp(x - torch.where(lse == -math.inf, 0.0, lse))
            del x
            o = p @ vh
            part(out, rq, h).copy_(o)
            if train:
                g = part(do, rq, h)
                part(dv, rk, h // group).add_(p.T @ g)
                x = p * (g @ vh.T - (g * o).sum(-1, keepdim=True))
                part(dq, rq, h).copy_(x @ kh * scale)
                part(dk, rk, h // group).add_(x.T @ qh * scale)
                dtable[:, h] += torch.bincount(which.flatten(), weights=x.flatten(), minlength=case["buckets"])
    return [out, dq, dk, dv, dtable] if train else out
