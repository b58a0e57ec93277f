"""Cases, inputs and plain forms of the operators that a language-model layer is made of.

Beside the DiT the framework runs two language models: the umT5 text encoder and the reward
model's backbone.  Three operators make up a layer of either:

  attend   ``ops.packed_attention`` / ``Fn.packed_attention``: attention inside packed sequences of
           different lengths, causal or not, grouped heads, queries that are the last tokens of
           their keys, a bias by relative position; with log-sum-exp, or with its gradients
  ffn      ``Fn.gated_ffn``: act(x Wg^T) * (x Wu^T) and the down projection, or its training step
  rotary   ``ops.rotary`` / ``Fn.rotary``: rotation of q and k by position tables, interleaved or
           half layout, part of the head, one position or several axes, scaled tables

Conventions.  Sequence s owns rows start[s] .. start[s] + length[s] of q and of k, v.  Query i of a
sequence with lq queries and lk keys stands at position i + lk - lq; causal queries see the keys up
to their position.  A query that sees no key gives zeros and a log-sum-exp of -inf.  The bias of
head h is ``rel_bias[h, key position - query position + M - 1]``, fp32 [H, 2 M - 1].  A rotary table
is fp32 [positions, R / 2, 2], cosine and sine of each pair's angle; pairs are (2 i, 2 i + 1) in
the interleaved layout and (i, i + R / 2) in the half layout, and elements from R on are copied.
"""
import math

import torch

own = False


def listed():
    return [
        # the conditional and the empty prompt of one video through the text encoder: latency counts
        {"name": "attend_two_prompts", "op": "attend", "mode": "forward", "seqs": 2, "shortest": 1, "longest": 77,
         "keys": 0, "heads": 64, "kv_heads": 64, "dim": 64, "causal": False, "bias": True, "fused": True},
        # prompts of a text-embedding batch, 20 to 512 tokens each, relative-position bias
        {"name": "attend_prompt_batch", "op": "attend", "mode": "forward", "seqs": 32, "shortest": 20, "longest": 512,
         "keys": 0, "heads": 64, "kv_heads": 64, "dim": 64, "causal": False, "bias": True, "fused": False},
        # a scoring batch of the reward model: video and text tokens of eight samples, grouped heads
        {"name": "attend_scoring", "op": "attend", "mode": "forward", "seqs": 8, "shortest": 600, "longest": 2500,
         "keys": 0, "heads": 12, "kv_heads": 2, "dim": 128, "causal": True, "bias": False, "fused": True},
        # one long prompt (an odd number of tokens), seven query heads to a key head
        {"name": "attend_long", "op": "attend", "mode": "forward", "seqs": 1, "shortest": 20161, "longest": 20161,
         "keys": 0, "heads": 28, "kv_heads": 4, "dim": 128, "causal": True, "bias": False, "fused": False},
        # one new token each for 48 sequences over what they hold already
        {"name": "attend_last_tokens", "op": "attend", "mode": "forward", "seqs": 48, "shortest": 1, "longest": 1,
         "keys": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "bias": False, "fused": False},
        # fine-tuning a reward backbone: packed samples of very different lengths, forward and backward
        {"name": "attend_train", "op": "attend", "mode": "train", "seqs": 12, "shortest": 5, "longest": 4096,
         "keys": 0, "heads": 16, "kv_heads": 4, "dim": 128, "causal": True, "bias": False, "fused": True},
        # one token through a text-encoder block: the weights are what is read
        {"name": "ffn_one_token", "op": "ffn", "mode": "forward", "tokens": 1, "in": 4096, "hidden": 10240,
         "act": "gelu_tanh"},
        # two prompts through the same block
        {"name": "ffn_two_prompts", "op": "ffn", "mode": "forward", "tokens": 154, "in": 4096, "hidden": 10240,
         "act": "gelu_tanh"},
        # training step of a gated block at the sizes of the 14B model's feed-forward, one of four SSP ranks
        {"name": "ffn_train", "op": "ffn", "mode": "train", "tokens": 20160, "in": 5120, "hidden": 13824, "act": "silu"},
        # one token of a reward backbone: launch latency counts
        {"name": "rotary_one_token", "op": "rotary", "mode": "forward", "tokens": 1, "heads": 12, "kv_heads": 2,
         "dim": 128, "rotate": 128, "layout": "half", "axes": 1, "dtype": "bfloat16", "scaled": False, "fused": True},
        # q and k of the 14B DiT at 81 frames of 768 x 1280: three axes (t, h, w), interleaved pairs
        {"name": "rotary_video", "op": "rotary", "mode": "forward", "tokens": 80640, "heads": 40, "kv_heads": 40,
         "dim": 128, "rotate": 128, "layout": "interleaved", "axes": 3, "dtype": "bfloat16", "scaled": False,
         "fused": False},
        # half of each head, far positions, scaled table, fp32, with gradients
        {"name": "rotary_train_part", "op": "rotary", "mode": "train", "tokens": 14039, "heads": 16, "kv_heads": 4,
         "dim": 128, "rotate": 64, "layout": "half", "axes": 1, "dtype": "float32", "scaled": True, "fused": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "ffn", "rotary"])
    mode = rng.choice(["forward", "train"])
    if op == "attend":
        kv = rng.choice([1, 2, 4, 8])
        c = {"op": op, "mode": mode, "seqs": _log(rng, 1, 64), "shortest": 0, "longest": _log(rng, 1, 12000), "keys": 0,
             "heads": kv * rng.choice([1, 2, 3, 4, 6, 7, 8]), "kv_heads": kv, "dim": rng.choice([40, 64, 80, 96, 128, 128]),
             "causal": rng.random() < 0.7, "bias": False, "fused": rng.random() < 0.5}
        c["shortest"] = _log(rng, 1, c["longest"])
        kind = rng.random()
        if kind < 0.3:                     # the last tokens of longer sequences
            c.update(mode="forward", longest=_log(rng, 1, 32), shortest=1, keys=_log(rng, 1, 12000))
        elif kind < 0.5:                   # a text encoder
            c.update(mode="forward", longest=min(c["longest"], 1024), shortest=min(c["shortest"], 1024), causal=False,
                     bias=True, dim=64)
        passes = 14 if c["mode"] == "train" else 4
        while passes * c["dim"] * c["heads"] * c["seqs"] * c["longest"] * max(c["longest"], c["keys"]) > 2.5e12:
            if c["seqs"] > 1:
                c["seqs"] = (c["seqs"] + 1) // 2
            else:
                c["longest"] = c["longest"] * 3 // 4
            c["shortest"] = min(c["shortest"], c["longest"])
        return c
    if op == "ffn":
        c = {"op": op, "mode": mode, "tokens": _log(rng, 1, 20160), "in": 8 * _log(rng, 16, 640),
             "hidden": 8 * _log(rng, 32, 1728), "act": rng.choice(["silu", "gelu_tanh"])}
        return c
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 80, 96, 128, 256])
    axes = rng.choice([1, 1, 3])
    return {"op": op, "mode": mode, "tokens": _log(rng, 1, 80640), "heads": kv * rng.choice([1, 2, 4, 5]), "kv_heads": kv,
            "dim": dim, "rotate": dim if rng.random() < 0.6 else 8 * rng.randint(1, dim // 8),
            "layout": rng.choice(["half", "interleaved"]), "axes": axes,
            "dtype": rng.choice(["bfloat16", "float16", "float32"]), "scaled": rng.random() < 0.4,
            "fused": rng.random() < 0.5}


# ---------------------------------------------------------------------------- inputs

def _lengths(case):
    """(queries, keys) of each sequence: spread evenly over the logarithm, the longest among them,
    in an order that is neither rising nor falling.  They belong to the case, not to the seed."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]

    def spread(lo, hi, step):
        v = [round(math.exp(math.log(max(lo, 1)) + (math.log(hi) - math.log(max(lo, 1))) * i / max(n - 1, 1)))
             for i in range(n)]
        v[-1] = hi
        return [v[(i * step + n - 1) % n] for i in range(n)]
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    lq = spread(lo, hi, step)
    if not case["keys"]:
        return lq, lq
    return lq, spread(max(1, case["keys"] // 8), case["keys"], next(s for s in (11, 9, 5, 1) if math.gcd(s, n) == 1))


def _pairs(case):
    """Allowed (query, key) pairs of one head."""
    total = 0
    for a, b in zip(*_lengths(case)):
        if not case["causal"]:
            total += a * b
        else:                             # query i sees max(0, i + 1 + b - a) keys
            first = max(1, b - a + 1)
            total += (first + b) * (b - first + 1) // 2
    return total


def _split(x, sizes):
    """Views [n, heads, dim] of the columns of a fused projection [n, sum of heads x dim]."""
    return [t.unflatten(1, (-1, sizes[0])) for t in x.split([sizes[0] * h for h in sizes[1:]], 1)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)

    s = {"case": case}
    if case["op"] == "attend":
        lq, lk = _lengths(case)
        h, kv, d = case["heads"], case["kv_heads"], case["dim"]
        if case["fused"] and not case["keys"]:          # views of one projection
            s["q"], s["k"], s["v"] = _split(normal(sum(lq), (h + 2 * kv) * d), (d, h, kv, kv))
        else:
            s["q"], s["k"], s["v"] = normal(sum(lq), h, d), normal(sum(lk), kv, d), normal(sum(lk), kv, d)
        s["scale"] = d ** -0.5
        if case["bias"]:                                # the text encoder scales no scores: its weights do
            m = max(lq)
            s["q"] = s["q"].mul(0.125)
            s["scale"] = 1.0
            far = torch.arange(1 - m, m, device="cuda").abs().float()
            s["rel_bias"] = torch.randn(h, 2 * m - 1, generator=g, device="cuda") - torch.log1p(far) * 0.3
        if case["mode"] == "train":
            s["do"] = normal(*s["q"].shape)
            for n in "qkv":
                s[n] = s[n].detach().requires_grad_(True)
        s["lq"], s["lk"] = lq, lk
        if own:
            from osp_next_b200 import ops
            s["pack"] = ops.SequencePack(lq, lk if case["keys"] else None, device="cuda")
        return s
    if case["op"] == "ffn":
        m, k, f = case["tokens"], case["in"], case["hidden"]
        s["x"] = normal(m, k)
        s["wg"], s["wu"], s["wd"] = normal(f, k, std=k ** -0.5), normal(f, k, std=k ** -0.5), normal(k, f, std=f ** -0.5)
        if case["mode"] == "train":
            s["dy"] = normal(m, k)
            for n in ("x", "wg", "wu", "wd"):
                s[n].requires_grad_(True)
        return s
    n, h, kv, d, r = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rotate"]
    dtype = getattr(torch, case["dtype"])
    if case["fused"]:
        s["q"], s["k"] = _split(normal(n, (h + 2 * kv) * d, dtype=dtype), (d, h, kv, kv))[:2]
    else:
        s["q"], s["k"] = normal(n, h, d, dtype=dtype), normal(n, kv, d, dtype=dtype)
    # one axis: a stretch of a context 20 times as long; three: frames of 48 x 80 tokens
    s["positions"] = max(1024, 20 * n) if case["axes"] == 1 else 1024
    at = torch.arange(n, device="cuda", dtype=torch.int32)
    if case["axes"] > 1:
        at = torch.stack([at // 3840, at // 80 % 48, at % 80], 1)
    s["pos"] = at + torch.randint(0, 900 if case["axes"] > 1 else s["positions"] - n + 1, (), generator=g, device="cuda",
                                  dtype=torch.int32)
    s["sections"] = None if case["axes"] == 1 else (r // 2 - 2 * (r // 6), r // 6, r // 6)
    s["angle"] = _inverse_wavelengths(case).cuda()
    a = torch.arange(s["positions"], device="cuda", dtype=torch.float64)[:, None] * s["angle"]
    s["table"] = torch.stack([a.cos(), a.sin()], -1).mul_(_magnitude(case)).float()
    if case["mode"] == "train":
        s["dq"], s["dk"] = normal(n, h, d, dtype=dtype), normal(n, kv, d, dtype=dtype)
        for t in "qk":
            s[t] = s[t].detach().requires_grad_(True)
    return s


SCALE, TRAINED, FAST, SLOW = 8.0, 4096, 32.0, 1.0      # context 8 times that of training


def _inverse_wavelengths(case):
    """Angle of pair i per position, in 64 bits.  Scaled: pairs that turn less than SLOW times within
    the trained length are slowed by SCALE, those of more than FAST turns are kept, linear between."""
    r = case["rotate"]
    f = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if not case["scaled"]:
        return f

    def pair(turns):
        return r * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
    lo, hi = max(math.floor(pair(FAST)), 0), min(math.ceil(pair(SLOW)), r - 1)
    slow = ((torch.arange(r // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f * (1 - slow) + f / SCALE * slow


def _magnitude(case):
    return 0.1 * math.log(SCALE) + 1.0 if case["scaled"] else 1.0


# ---------------------------------------------------------------------------- one pass

def run(s):
    return _RUN[s["case"]["op"]](s)


def _chunks(s):
    """Runs of sequences that are padded to one batch, and the key heads taken at once: at most
    2^29 scores at a time."""
    c, most = s["case"], 1 << 29
    group = c["heads"] // c["kv_heads"]
    one = [a * b for a, b in zip(s["lq"], s["lk"])]
    first = 0
    while first < c["seqs"]:
        last, a, b = first + 1, s["lq"][first], s["lk"][first]
        while last < c["seqs"]:
            na, nb = max(a, s["lq"][last]), max(b, s["lk"][last])
            if (last + 1 - first) * na * nb * c["heads"] > min(most, 2 * c["heads"] * (sum(one[first:last + 1]) + (1 << 14))):
                break
            a, b, last = na, nb, last + 1
        at_once = max(1, min(c["kv_heads"], most // max(1, (last - first) * a * b * group)))
        for h in range(0, c["kv_heads"], at_once):
            yield first, last, h, min(c["kv_heads"], h + at_once)
        first = last


def _rows(lengths, first, last, device):
    """Row of each (sequence, place) of a padded batch, -1 where there is none."""
    n = torch.tensor(lengths[first:last])[:, None]
    start = torch.tensor([sum(lengths[:first])] + lengths[first:last - 1]).cumsum(0)[:, None]
    at = torch.arange(max(1, max(lengths[first:last])))[None]
    return torch.where(at < n, start + at, -1).to(device), n.to(device)


def _scores(s, first, last, h0, h1):
    """Padded q [S, G, A, D], k and v [S, G', B, D] in 32 bits, allowed scores and their mask."""
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    rq, nq = _rows(s["lq"], first, last, s["q"].device)
    rk, nk = _rows(s["lk"], first, last, s["q"].device)
    q = s["q"].detach()[rq.clamp(min=0), h0 * group:h1 * group].float().transpose(1, 2)
    k = s["k"].detach()[rk.clamp(min=0), h0:h1].float().transpose(1, 2)
    v = s["v"].detach()[rk.clamp(min=0), h0:h1].float().transpose(1, 2)
    q = q.unflatten(1, (h1 - h0, group)).flatten(2, 3)
    scores = (q @ k.transpose(2, 3)).mul_(s["scale"]).unflatten(2, (group, -1))
    at_q = torch.arange(rq.shape[1], device=rq.device)[None, :, None]
    at_k = torch.arange(rk.shape[1], device=rq.device)[None, None, :]
    off = (nk - nq)[:, :, None]
    if c["bias"]:
        m = (s["rel_bias"].shape[1] + 1) // 2
        places = (at_k - at_q - off + m - 1).clamp(0, 2 * m - 2)
        bias = s["rel_bias"][h0 * group:h1 * group][:, places].transpose(0, 1)
        scores += bias.unflatten(1, (h1 - h0, group))
    allowed = (at_q < nq[:, :, None]) & (at_k < nk[:, :, None])
    if c["causal"]:
        allowed = allowed & (at_k <= at_q + off)
    allowed = allowed[:, None, None]
    return rq, rk, q, k, v, scores.masked_fill_(~allowed, -math.inf), allowed


def _run_attend(s):
    c = s["case"]
    train = c["mode"] == "train"
    if own:
        if train:
            from osp_next_b200.models import functional as Fn
            o = Fn.packed_attention(s["q"], s["k"], s["v"], s["pack"], causal=c["causal"], scale=s["scale"])
            return [o.detach(), *torch.autograd.grad(o, [s["q"], s["k"], s["v"]], s["do"])]
        from osp_next_b200 import ops
        return ops.packed_attention(s["q"], s["k"], s["v"], s["pack"], causal=c["causal"], scale=s["scale"],
                                    rel_bias=s.get("rel_bias"), return_lse=True)
    group, dim = c["heads"] // c["kv_heads"], c["dim"]
    new = {"device": s["q"].device, "dtype": torch.bfloat16}
    o = torch.zeros(s["q"].shape, **new)
    lse = torch.full(s["q"].shape[:2], -math.inf, device=s["q"].device)
    dq, dk, dv = ([torch.zeros(s[n].shape, **new) for n in "qkv"] if train else (None, None, None))
    for first, last, h0, h1 in _chunks(s):
        rq, rk, q, k, v, scores, allowed = _scores(s, first, last, h0, h1)
        top = scores.amax(4, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
        p = scores.sub_(top).exp_()
        total = p.sum(4, keepdim=True)
        p.div_(total.clamp(min=1e-30))
        out = (p.flatten(2, 3) @ v).unflatten(2, (group, -1))
        real = rq >= 0
        heads = slice(h0 * group, h1 * group)

        def back(t):                       # [S, heads, group, A, D] -> rows [n, heads, D]
            return t.flatten(1, 2).transpose(1, 2)[real]
        o[rq[real], heads] = back(out).to(torch.bfloat16)
        lse[rq[real], heads] = back(top + torch.log(total))[..., 0]
        if train:
            do = s["do"][rq.clamp(min=0), heads].float().masked_fill_(~real[:, :, None, None], 0.0)
            do = do.transpose(1, 2).unflatten(1, (h1 - h0, group))
            seen = rk >= 0
            flat = p.flatten(2, 3)
            dv[rk[seen], h0:h1] = (flat.transpose(2, 3) @ do.flatten(2, 3)).transpose(1, 2)[seen].to(torch.bfloat16)
            dp = (do.flatten(2, 3) @ v.transpose(2, 3)).unflatten(2, (group, -1))
            ds = dp.sub_((do * out).sum(4, keepdim=True)).mul_(p).mul_(s["scale"]).flatten(2, 3)
            dk[rk[seen], h0:h1] = (ds.transpose(2, 3) @ q).transpose(1, 2)[seen].to(torch.bfloat16)
            dq[rq[real], heads] = back((ds @ k).unflatten(2, (group, -1))).to(torch.bfloat16)
    return [o, dq, dk, dv] if train else (o, lse)


def _act(g, kind):
    """act(g) and its derivative."""
    if kind == "silu":
        p = 1 / (1 + torch.exp(-g))
        return g * p, p * (1 + g * (1 - p))
    t = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g))
    inner = math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * inner


def _run_ffn(s):
    c = s["case"]
    train = c["mode"] == "train"
    if own:
        from osp_next_b200.models import functional as Fn
        y = Fn.gated_ffn(s["x"], s["wg"], s["wu"], s["wd"], act=c["act"])
        return [y.detach(), *torch.autograd.grad(y, [s["x"], s["wg"], s["wu"], s["wd"]], s["dy"])] if train else y
    x, wg, wu, wd = (s[n].detach().float() for n in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(g, c["act"])
    h = a * u
    y = (h @ wd.t()).to(torch.bfloat16)
    if not train:
        return y
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    return [y] + [t.to(torch.bfloat16) for t in (dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ h)]


def _run_rotary(s):
    c = s["case"]
    train = c["mode"] == "train"
    if own:
        kw = {"layout": c["layout"], "sections": s["sections"]}
        if train:
            from osp_next_b200.models import functional as Fn
            q, k = Fn.rotary(s["q"], s["k"], s["pos"], s["table"], **kw)
            return [q.detach(), k.detach(), *torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])]
        from osp_next_b200 import ops
        return ops.rotary(s["q"], s["k"], s["pos"], s["table"], **kw)
    r = c["rotate"]
    pos = s["pos"].double()
    if c["axes"] > 1:
        axis = torch.tensor([i for i, n in enumerate(s["sections"]) for _ in range(n)], device=pos.device)
        pos = pos[:, axis]
    else:
        pos = pos[:, None]
    angle = pos * s["angle"]
    cos = angle.cos().mul_(_magnitude(c)).float()[:, None]
    sin = angle.sin().mul_(_magnitude(c)).float()[:, None]

    def turn(x, sin):
        x = x.detach()
        y = x.float()
        if c["layout"] == "half":
            a, b = y[..., :r // 2], y[..., r // 2:r]
            z = torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., r:]], -1)
        else:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            z = torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), y[..., r:]], -1)
        return z.to(x.dtype)
    out = [turn(s["q"], sin), turn(s["k"], sin)]
    return out + [turn(s["dq"], -sin), turn(s["dk"], -sin)] if train else tuple(out)


_RUN = {"attend": _run_attend, "ffn": _run_ffn, "rotary": _run_rotary}


def work(case):
    if case["op"] == "attend":
        lq, lk = (sum(v) for v in _lengths(case))
        h, kv, d = case["heads"], case["kv_heads"], case["dim"]
        pairs = _pairs(case) * h
        if case["mode"] == "train":       # q, k, v, dO read; o, dq, dk, dv written
            return {"bytes": 2 * d * (4 * lq * h + 4 * lk * kv), "flops": 14 * d * pairs}
        bias = 4 * h * (2 * max(_lengths(case)[0]) - 1) if case["bias"] else 0
        return {"bytes": 2 * d * (2 * lq * h + 2 * lk * kv) + 4 * lq * h + bias, "flops": 4 * d * pairs}
    if case["op"] == "ffn":
        m, k, f = case["tokens"], case["in"], case["hidden"]
        if case["mode"] == "train":       # x, dy, weights read; y, dx, weight gradients written
            return {"bytes": 2 * (4 * m * k + 6 * k * f), "flops": 18 * m * k * f}
        return {"bytes": 2 * (2 * m * k + 3 * k * f), "flops": 6 * m * k * f}
    n, d, size = case["tokens"], case["dim"], 4 if case["dtype"] == "float32" else 2
    turns = 2 if case["mode"] == "train" else 1
    values = n * (case["heads"] + case["kv_heads"])
    return {"bytes": turns * (values * d * 2 * size) + n * (4 * case["rotate"] + 4 * case["axes"]),
            "flops": turns * values * case["rotate"] * 3}


# ---------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    if case["op"] == "ffn":
        x, wg, wu, wd = (s[n].detach().double().requires_grad_(case["mode"] == "train") for n in ("x", "wg", "wu", "wd"))
        g = x @ wg.t()
        gate = g * torch.sigmoid(g) if case["act"] == "silu" else \
            g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        y = (gate * (x @ wu.t())) @ wd.t()
        if case["mode"] != "train":
            return y
        return [y.detach(), *torch.autograd.grad(y, [x, wg, wu, wd], s["dy"].double())]
    r, axes = case["rotate"], case["axes"]
    pos = s["pos"].double().view(case["tokens"], axes)
    counts = torch.tensor(s["sections"] if axes > 1 else [r // 2], device=pos.device)
    angle = pos.repeat_interleave(counts, 1) * s["angle"]
    turn = torch.polar(torch.full_like(angle, _magnitude(case)), angle)[:, None]

    def rotated(x, turn):
        x = x.detach().double()
        head = x[..., :r]
        pairs = head.unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" else \
            head.unflatten(-1, (r // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.transpose(-1, -2) if case["layout"] == "half" else z
        return torch.cat([z.flatten(-2), x[..., r:]], -1)
    out = [rotated(s["q"], turn), rotated(s["k"], turn)]
    if case["mode"] == "train":
        return out + [rotated(s["dq"], turn.conj()), rotated(s["dk"], turn.conj())]
    return tuple(out)


def _exact_attend(case, s):
    """One sequence and query head after the other, blocks of queries at a time."""
    group = case["heads"] // case["kv_heads"]
    q, k, v = (s[n].detach() for n in "qkv")
    train = case["mode"] == "train"
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)] if train else []
    a0 = b0 = 0
    for a, b in zip(s["lq"], s["lk"]):
        key = torch.arange(b, device=q.device)
        step = max(1, (1 << 26) // max(1, b * group))
        for i in range(0, a if b else 0, step):
            rows = slice(a0 + i, a0 + min(a, i + step))
            place = torch.arange(i, min(a, i + step), device=q.device) + b - a
            seen = key[None] <= place[:, None] if case["causal"] else None
            for h in range(case["kv_heads"]):
                hs = slice(h * group, (h + 1) * group)
                qh, kh, vh = q[rows, hs].double(), k[b0:b0 + b, h].double(), v[b0:b0 + b, h].double()
                z = torch.einsum("nhd,kd->hnk", qh, kh) * s["scale"]
                if case["bias"]:
                    m = (s["rel_bias"].shape[1] + 1) // 2
                    z = z + s["rel_bias"][hs].double()[:, key[None] - place[:, None] + m - 1]
                if seen is not None:
                    z = torch.where(seen, z, -math.inf)
                l = torch.logsumexp(z, -1)
                w = torch.where(torch.isinf(l)[..., None], 0.0, torch.exp(z - l[..., None]))
                lse[rows, hs] = l.t()
                out = torch.einsum("hnk,kd->nhd", w, vh)
                o[rows, hs] = out
                if train:
                    do = s["do"][rows, hs].double()
                    grads[2][b0:b0 + b, h] += torch.einsum("hnk,nhd->kd", w, do)
                    dz = w * (torch.einsum("nhd,kd->hnk", do, vh) - (do * out).sum(-1).t()[..., None]) * s["scale"]
                    grads[0][rows, hs] = torch.einsum("hnk,kd->nhd", dz, kh)
                    grads[1][b0:b0 + b, h] += torch.einsum("hnk,nhd->kd", dz, qh)
        a0, b0 = a0 + a, b0 + b
    return [o, *grads] if train else (o, lse)
