"""Attention over packed sequences: work lists and refusals on the CPU, kernels against the formula in
64 bits.  Bounds count roundings: half a bf16 step is 2^-8 of a value, P and dS are rounded to bf16
before their products, results once more; sums run in fp32 (2^-23 a term, the tensor core cuts)."""
import math

import numpy as np
import pytest
import torch

from osp_next_b200 import ops
from osp_next_b200.models import functional as Fn
from osp_next_b200.ops import packed

HALF = 2.0 ** -8           # half a bf16 step
F32 = 2.0 ** -23


def oracle(q, k, v, pack, causal, scale, bias=None, do=None):
    """Values in 64 bits and, for each, the largest error that the roundings allow."""
    q, k, v = q.double(), k.double(), v.double()
    group = q.shape[1] // k.shape[1]
    D = q.shape[2]
    out = {"o": torch.zeros_like(q), "eo": torch.zeros_like(q),
           "lse": torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device),
           "else": torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)}
    if do is not None:
        do = do.double()
        out.update({n: torch.zeros_like(t) for n, t in (("dq", q), ("edq", q), ("dk", k), ("edk", k), ("dv", v),
                                                        ("edv", v))})
    for a0, a, b0, b in zip(pack.starts, pack.lengths, pack.key_starts, pack.key_lengths):
        for h in range(q.shape[1] if a and b else 0):
            g = h // group
            qs, ks, vs = q[a0:a0 + a, h], k[b0:b0 + b, g], v[b0:b0 + b, g]
            s = qs @ ks.t() * scale
            es = (D + 2) * F32 * abs(scale) * (qs.abs() @ ks.abs().t()) + 4 * F32 * s.abs()
            place = torch.arange(b - a, b, device=q.device)[:, None]
            key = torch.arange(b, device=q.device)[None]
            if bias is not None:
                add = bias.double()[h][key - place + (bias.shape[1] + 1) // 2 - 1]
                s = s + add
                es = es + 4 * F32 * (add.abs() + s.abs())
            seen = key <= place if causal else torch.ones_like(s, dtype=torch.bool)
            s = s.masked_fill(~seen, -math.inf)
            es = es.masked_fill(~seen, 0.0)
            lse = torch.logsumexp(s, 1)
            p = torch.where(torch.isinf(lse)[:, None], 0.0, torch.exp(s - lse[:, None]))
            # a weight is off by exp(2 max es) - 1 (its own score and the sum), 2^-22 of the exponential
            # and 2^-23 for each term of the row sum
            off = (2 * es.amax(1, keepdim=True) + 16 * F32 + F32 * b ** 0.5 * 4).expm1()
            o = p @ vs
            eo = HALF * o.abs() + (1 + HALF) * (HALF + off) * (p @ vs.abs()) + b * F32 * (p @ vs.abs())
            out["o"][a0:a0 + a, h], out["eo"][a0:a0 + a, h] = o, eo
            out["lse"][a0:a0 + a, h] = lse
            out["else"][a0:a0 + a, h] = es.amax(1) + 16 * F32 + 4 * F32 * torch.where(torch.isinf(lse), 0.0, lse).abs() \
                + 4 * F32 * torch.where(seen.any(1), s.masked_fill(~seen, 0.0).abs().amax(1), 0.0)
            if do is None:
                continue
            dos = do[a0:a0 + a, h]
            offp = off + out["else"][a0:a0 + a, h][:, None] * 2
            out["dv"][b0:b0 + b, g] += p.t() @ dos
            out["edv"][b0:b0 + b, g] += ((HALF + offp) * p).t() @ dos.abs() + a * F32 * (p.t() @ dos.abs())
            dp = dos @ vs.t()
            delta = (dos * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            e = p * ((dos.abs() * (eo + HALF * o.abs())).sum(1, keepdim=True) + D * F32 * (dos.abs() @ vs.abs().t())
                     + D * F32 * (dos * o).abs().sum(1, keepdim=True)) + (HALF + offp) * ds.abs()
            e = e * (1 + HALF)
            out["dq"][a0:a0 + a, h] = ds @ ks * scale
            out["edq"][a0:a0 + a, h] = (e @ ks.abs() + b * F32 * (ds.abs() @ ks.abs())) * scale
            out["dk"][b0:b0 + b, g] += ds.t() @ qs * scale
            out["edk"][b0:b0 + b, g] += (e.t() @ qs.abs() + a * F32 * (ds.abs().t() @ qs.abs())) * scale
    if do is not None:
        for n in ("dq", "dk", "dv"):
            out["e" + n] = out["e" + n] * (1 + HALF) + HALF * out[n].abs()
    return out


def close(got, want, err, what):
    got = got.double()
    assert got.shape == want.shape, what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what + ": infinities"
    d = (got - want).abs()[~inf]
    assert not torch.isnan(d).any(), what + ": NaN"
    worst = (d - err[~inf]).max().item() if d.numel() else -1.0
    assert worst <= 1e-30, f"{what}: {worst:.3g} over the bound (largest error {d.max().item():.3g})"


def tensors(pack, heads, kv_heads, dim, device, seed=0, dtype=torch.bfloat16, spare=0, std=1.0):
    g = torch.Generator(device=device).manual_seed(seed)

    def rand(n, h):
        return (torch.randn(n + spare, h, dim, generator=g, device=device) * std).to(dtype)
    return rand(pack.rows, heads), rand(pack.key_rows, kv_heads), rand(pack.key_rows, kv_heads), rand(pack.rows, heads)


# ---------------------------------------------------------------------------- CPU

PACKS = [([1], None), ([1, 1, 1], None), ([128], None), ([127, 1, 129], None), ([5, 0, 300, 77], None),
         ([1, 3, 130], [700, 3, 131]), ([9, 4, 200], [2, 0, 130]), ([0, 0], None), ([], None), ([1], [3000])]


@pytest.mark.parametrize("lengths,keys", PACKS)
@pytest.mark.parametrize("group,kv", [(1, 3), (3, 2), (7, 1), (40, 1), (128, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_work_lists_cover_every_pair_once(lengths, keys, group, kv, causal):
    """What the kernels would compute from the lists: every allowed (query, key) pair of a sequence
    once forward, once for dQ and once for dK, dV; every row written by one item or one join."""
    pack = ops.SequencePack(lengths, keys, device="cpu")
    per, T = 128 // group, 128
    seq_of = np.repeat(np.arange(len(pack)), pack.lengths)
    want = np.zeros((pack.rows, pack.key_rows), dtype=int)
    for s in range(len(pack)):
        a0, a, b0, b = pack.starts[s], pack.lengths[s], pack.key_starts[s], pack.key_lengths[s]
        i, j = np.arange(a)[:, None], np.arange(b)[None]
        want[a0:a0 + a, b0:b0 + b] = (j <= i + b - a) if causal else 1

    def mark(seen, row, n_q, limit, k_row, n_keys, kt0, kt1):
        for i in range(n_q):
            lim = min(n_keys, limit + i) if causal else n_keys
            cols = np.arange(kt0 * T, min(kt1 * T, max(lim, 0)))
            seen[row + i, k_row + cols] += 1

    for sms, tiles in ((1, 2), (4, 1), (148, 2), (148, 1), (4000, 2), (4000, 1)):
        (items, joins), slots = packed.forward_items(pack, group, kv, causal, sms, tiles)
        seen, written = np.zeros_like(want), np.zeros(pack.rows, dtype=int)
        used = []
        for row, n_q, limit, k_row, n_keys, kt0, kt1, slot in items:
            assert 0 < n_q <= tiles * packed.positions(pack, group) <= tiles * per and (kt1 > kt0 or kt0 == 0 == kt1) and kt1 <= -(-n_keys // T)
            assert len(set(seq_of[row:row + n_q])) == 1
            mark(seen, row, n_q, limit, k_row, n_keys, kt0, kt1)
            if slot < 0:
                written[row:row + n_q] += 1
            else:
                used.append(slot)
        for row, n_q, first, parts in joins:
            assert parts > 1
            mine = sorted(tuple(x) for x in items if x[7] >= first and x[7] < first + parts)
            assert len(mine) == parts and all(x[0] == row and x[1] == n_q for x in mine)
            written[row:row + n_q] += 1
        assert sorted(used) == list(range(slots))
        assert np.array_equal(seen, want) and np.all(written == 1)
        assert np.all(np.diff(items[:, 6] - items[:, 5]) <= 0)

        items, joins, slots = packed.key_items(pack, group, kv, causal, sms)
        seen, written, used = np.zeros_like(want), np.zeros(pack.key_rows, dtype=int), []
        for k_row, n_k, first, q_row, n_q, lead, slot, _ in items:
            assert 0 < n_k <= T and n_q >= 0
            for r in range(n_k):
                rows = np.arange(max(0, lead + r) if causal else 0, n_q)
                seen[q_row + rows, k_row + r] += 1
            if slot < 0:
                written[k_row:k_row + n_k] += 1
            else:
                used.append(slot)
        for k_row, n_k, first, parts in joins:
            written[k_row:k_row + n_k] += 1
            assert parts > 1
        assert sorted(used) == list(range(slots)) and sum(joins[:, 3]) == slots
        assert np.array_equal(seen, want) and np.all(written == 1)

    seen = np.zeros_like(want)
    for row, n_q, limit, k_row, n_keys, kt0, kt1, slot in packed.row_items(pack, group, causal):
        assert 0 < n_q <= per and kt0 == 0 and slot == -1
        mark(seen, row, n_q, limit, k_row, n_keys, kt0, kt1)
    assert np.array_equal(seen, want)


@pytest.mark.parametrize("causal", [True, False])
def test_reference_against_64_bits_and_differences(causal):
    pack = ops.SequencePack([3, 1, 5], [3, 4, 2], device="cpu")
    q, k, v, do = tensors(pack, 4, 2, 8, "cpu", dtype=torch.float64)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    assert torch.autograd.gradcheck(lambda *t: Fn.packed_attention(*t, pack, causal=causal), leaves)
    want = oracle(*[t.detach() for t in leaves], pack, causal, 8 ** -0.5, do=do)
    with torch.no_grad():
        o, lse = ops.packed_attention(q, k, v, pack, causal=causal, return_lse=True)
    assert torch.allclose(o, want["o"], atol=1e-12) and torch.allclose(lse, want["lse"], atol=1e-12)
    for got, n in zip(packed.packed_attention_bwd(*[t.detach() for t in leaves], o, do, lse, pack, causal),
                      ("dq", "dk", "dv")):
        assert torch.allclose(got, want[n], atol=1e-12)


def test_padded_pack_leaves_other_rows_zero():
    pack = ops.SequencePack.padded([2, 0, 4], 5, device="cpu")
    assert pack.starts.tolist() == [0, 5, 10] and pack.rows == 14 and not pack.dense
    q, k, v, _ = tensors(pack, 2, 2, 8, "cpu", dtype=torch.float32, spare=1)
    for t in (q, k, v):
        t[2:10] = math.nan
    o, lse = ops.packed_attention(q, k, v, pack, return_lse=True)
    rest = torch.ones(15, dtype=torch.bool)
    rest[[0, 1, 10, 11, 12, 13]] = False
    assert torch.isfinite(o).all() and (o[rest] == 0).all() and torch.isinf(lse[rest]).all()
    assert torch.isfinite(lse[~rest]).all()


def test_hidden_values_do_not_reach_a_row():
    pack = ops.SequencePack([4], device="cpu")
    q, k, v, _ = tensors(pack, 1, 1, 8, "cpu", dtype=torch.float32)
    want = ops.packed_attention(q, k, v, pack)
    v[2, 0, 3] = math.inf
    got = ops.packed_attention(q, k, v, pack)
    assert torch.equal(got[:2], want[:2]) and not torch.isfinite(got[2:, 0, 3]).any()


def test_refusals():
    P = ops.SequencePack
    with pytest.raises(TypeError, match="whole numbers"):
        P([1.5], device="cpu")
    with pytest.raises(TypeError, match="whole numbers"):
        P(torch.tensor([1.0]), device="cpu")
    with pytest.raises(ValueError, match="from 0"):
        P([3, -1], device="cpu")
    with pytest.raises(ValueError, match="overlap"):
        P([3, 3], starts=[0, 2], device="cpu")
    with pytest.raises(ValueError, match="2 lengths, 1 key_lengths"):
        P([3, 3], [3], device="cpu")
    with pytest.raises(ValueError, match="without key_lengths"):
        P([3], key_starts=[0], device="cpu")
    with pytest.raises(ValueError, match="rows of 4"):
        P.padded([5], 4, device="cpu")
    pack = P([3, 2], device="cpu")
    q, k, v, _ = tensors(pack, 4, 2, 16, "cpu", dtype=torch.float32)
    call = ops.packed_attention
    with pytest.raises(TypeError, match="SequencePack"):
        call(q, k, v, [3, 2])
    with pytest.raises(ValueError, match="needs 5 query"):
        call(q[:4], k, v, pack)
    with pytest.raises(ValueError, match="needs 5 query and 5 key"):
        call(q, k[:3], v[:3], pack)
    with pytest.raises(ValueError, match="3 query heads"):
        call(q[:, :3], k, v, pack)
    with pytest.raises(ValueError, match="head_dim"):
        call(q[..., :12], k[..., :12], v[..., :12], pack)
    with pytest.raises(ValueError, match=r"\[tokens, heads, head_dim\]"):
        call(q[None], k, v, pack)
    with pytest.raises(ValueError, match="against q"):
        call(q, k, v[:, :1], pack)
    with pytest.raises(TypeError, match="one type"):
        call(q, k.double(), v, pack)
    with pytest.raises(ValueError, match=r"rel_bias \[4"):
        call(q, k, v, pack, rel_bias=torch.zeros(4, 4))
    with pytest.raises(ValueError, match="reaches 2 positions"):
        call(q, k, v, pack, rel_bias=torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match="no gradient"):
        call(q.requires_grad_(), k, v, pack)
    with torch.no_grad():
        call(q, k, v, pack)
    big = ops.SequencePack([5], device="cpu")
    with pytest.raises(ValueError, match="needs 5"):
        Fn.packed_attention(q[:4], k[:4], v[:4], big)


# ---------------------------------------------------------------------------- GPU

gpu = pytest.mark.gpu
HEADS = [(4, 4, 64), (7, 1, 128), (6, 2, 80), (16, 2, 128), (40, 1, 40), (5, 1, 96), (2, 2, 8), (128, 1, 64)]


@pytest.fixture(params=[1, 2], ids=["one_tile", "two_tiles"])
def tiles(request, monkeypatch):
    """Both forms of the forward kernel at every size."""
    monkeypatch.setattr(packed, "row_tiles", lambda *a: request.param)


def _pass(pack, heads, kv, dim, causal, seed=0, bias=None, train=True, scale=None, std=1.0):
    q, k, v, do = tensors(pack, heads, kv, dim, "cuda", seed, std=std)
    scale = dim ** -0.5 if scale is None else scale
    want = oracle(q, k, v, pack, causal, scale, bias, do if train else None)
    o, lse = ops.packed_attention(q, k, v, pack, causal=causal, scale=scale, rel_bias=bias, return_lse=True)
    close(o, want["o"], want["eo"], "o")
    close(lse, want["lse"], want["else"], "lse")
    if train:
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        out = Fn.packed_attention(*leaves, pack, causal=causal, scale=scale)
        assert torch.equal(out, o)
        for g, n in zip(torch.autograd.grad(out, leaves, do), ("dq", "dk", "dv")):
            close(g, want[n], want["e" + n], n)
    ops.check_device_errors()


@gpu
@pytest.mark.parametrize("lengths,keys", PACKS)
@pytest.mark.parametrize("causal", [True, False])
def test_gpu_lengths(lengths, keys, causal, tiles):
    for heads, kv, dim in ((4, 2, 64), (6, 2, 128)):
        _pass(ops.SequencePack(lengths, keys), heads, kv, dim, causal)


@gpu
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("causal", [True, False])
def test_gpu_heads(heads, kv, dim, causal, tiles):
    _pass(ops.SequencePack([1, 150, 33, 0, 260]), heads, kv, dim, causal)


@gpu
def test_gpu_long_and_split(tiles):
    _pass(ops.SequencePack([2111, 5, 640]), 8, 2, 128, True)
    _pass(ops.SequencePack([1, 2, 40], [5003, 1200, 6001]), 8, 1, 128, True)
    _pass(ops.SequencePack([1], [9001]), 4, 4, 64, False)
    _pass(ops.SequencePack([3000]), 2, 1, 64, True)


@gpu
@pytest.mark.parametrize("lengths", [[1], [77, 3], [128, 129, 1, 512], [20, 200]])
def test_gpu_relative_bias(lengths, tiles):
    pack = ops.SequencePack(lengths)
    for extra in (0, 13):
        m = pack.longest + extra
        bias = torch.randn(8, 2 * m - 1, generator=torch.Generator("cuda").manual_seed(3), device="cuda") * 2
        _pass(pack, 8, 8, 64, False, bias=bias, train=False, scale=1.0, std=0.4)
        _pass(pack, 8, 2, 128, True, bias=bias, train=False, scale=0.05)
    _pass(ops.SequencePack([3, 4], [40, 200]), 4, 2, 64, True, bias=torch.randn(4, 399, device="cuda"), train=False)


@gpu
def test_gpu_large_scores(tiles):
    """Scores to some 500: the running maximum moves, weights are nearly one-hot."""
    _pass(ops.SequencePack([300, 41]), 4, 2, 64, True, std=6.0)


@gpu
def test_gpu_neighbours_and_gaps(tiles):
    """NaN and infinities in other sequences and in rows of none reach nobody."""
    pack = ops.SequencePack([70, 130, 5], starts=[3, 100, 240])
    q, k, v, do = tensors(pack, 6, 2, 64, "cuda", spare=4)
    clean = [t.clone() for t in (q, k, v, do)]
    rest = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    for a, n in zip(pack.starts, pack.lengths):
        rest[a:a + n] = False
    for t in (q, k, v, do):
        t[rest] = math.nan
        t[100:230] = math.inf                     # the second sequence itself
    for causal in (True, False):
        def run(q, k, v, do):
            leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
            o = Fn.packed_attention(*leaves, pack, causal=causal)
            with torch.no_grad():
                _, lse = ops.packed_attention(q, k, v, pack, causal=causal, return_lse=True)
            return [o.detach(), lse, *torch.autograd.grad(o, leaves, do)]
        want, got = run(*clean), run(q, k, v, do)
        for i, (w, g) in enumerate(zip(want, got)):
            for rows in (slice(3, 73), slice(240, 245)):
                assert torch.equal(w[rows], g[rows]), i
            blank = g[rest]
            assert (torch.isinf(blank) if i == 1 else blank == 0).all(), i
        assert torch.isnan(got[0][100:230]).all()


@gpu
def test_gpu_views_copies_and_devices():
    pack = ops.SequencePack([60, 90])
    qkv = torch.randn(150, 8 * 64, device="cuda").bfloat16()
    q, k, v = (t.unflatten(1, (-1, 64)) for t in qkv.split([256, 128, 128], 1))
    want = ops.packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), pack)
    assert torch.equal(ops.packed_attention(q, k, v, pack), want)
    wide = torch.zeros(150, 4, 65, device="cuda", dtype=torch.bfloat16)          # rows at odd addresses
    wide[..., 1:] = q
    assert torch.equal(ops.packed_attention(wide[..., 1:], k, v, pack), want)
    one = k[:, :1].expand(150, 2, 64)                                            # broadcast heads
    assert torch.equal(ops.packed_attention(q, one, one, pack),
                       ops.packed_attention(q, one.contiguous(), one.contiguous(), pack))
    leaf = k[:, :1].detach().clone().requires_grad_(True)
    o = Fn.packed_attention(q, leaf.expand(150, 2, 64), leaf.expand(150, 2, 64), pack)
    g, = torch.autograd.grad(o.sum(), leaf)
    w = oracle(q, one, one, pack, True, 0.125, do=torch.ones_like(q))
    close(g, (w["dk"] + w["dv"]).sum(1, keepdim=True), (w["edk"] + w["edv"]).sum(1, keepdim=True) * (1 + 3 * HALF)
          + 3 * HALF * (w["dk"].abs() + w["dv"].abs()).sum(1, keepdim=True), "broadcast gradient")
    with pytest.raises(TypeError, match="bf16"):
        ops.packed_attention(q.half(), k.half(), v.half(), pack)
    with pytest.raises(ValueError, match="pack on cpu"):
        ops.packed_attention(q, k, v, ops.SequencePack([60, 90], device="cpu"))
    f = Fn.packed_attention(q.float().requires_grad_(), k.float(), v.float(), pack)
    assert f.dtype == torch.bfloat16 and torch.equal(f, want)
    bias = torch.zeros(4, 179, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient with rel_bias"):
        Fn.packed_attention(q.detach().requires_grad_(), k, v, pack, rel_bias=bias)


@gpu
def test_gpu_offsets_past_32_bits():
    """Rows whose elements lie beyond 2^31 of their tensors: the same values as in a tensor of their own."""
    rows, heads, dim = 280000, 64, 128
    small = ops.SequencePack([130, 7])
    q, k, v, do = tensors(small, heads, 2, dim, "cuda")
    far = ops.SequencePack([130, 7], [130, 7], starts=[rows - 200, rows - 40], key_starts=[0, 130])
    big = []
    for t in (q, do):
        b = torch.zeros(rows, heads, dim, device="cuda", dtype=torch.bfloat16)
        b[rows - 200:rows - 70], b[rows - 40:rows - 33] = t[:130], t[130:]
        big.append(b)
    assert big[0].numel() > 1 << 31
    def run(q, k, v, do, pack):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = Fn.packed_attention(*leaves, pack)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]
    want, got = run(q, k, v, do, small), run(big[0], k, v, big[1], far)
    for w, g in ((want[0], got[0]), (want[1], got[1])):
        assert torch.equal(g[rows - 200:rows - 70], w[:130]) and torch.equal(g[rows - 40:rows - 33], w[130:])
        assert not g[:1000].any() and not g[rows - 70:rows - 40].any()
    assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])


@gpu
def test_gpu_two_streams_share_a_pack():
    """Calls of one pack on two streams at once, the pack dropped while they run."""
    packs = [ops.SequencePack([500, 1, 300]) for _ in range(2)]
    q, k, v, do = tensors(packs[0], 16, 4, 128, "cuda")
    want = ops.packed_attention(q, k, v, packs[0])
    ops.packed_attention(q, k, v, packs[1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.packed_attention(q, k, v, packs[1]))
    del packs[1]
    junk = [torch.full((64, 8), -1, dtype=torch.int32, device="cuda") for _ in range(50)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got) and len(junk) == 50


@gpu
def test_gpu_graph_streams_and_repeats():
    pack = ops.SequencePack([200, 31], [900, 31])
    q, k, v, do = tensors(pack, 8, 2, 128, "cuda")
    want = ops.packed_attention(q, k, v, pack)
    wantg = packed.packed_attention_bwd(q, k, v, *_with_lse(q, k, v, do, pack), pack)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.packed_attention(q, k, v, pack)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want)
    graphs = []
    for _ in range(2):                                     # two graphs on one pack
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, lse = ops.packed_attention(q, k, v, pack, return_lse=True)
            grads = packed.packed_attention_bwd(q, k, v, o, do, lse, pack)
        graphs.append((g, o, grads))
    for g, o, grads in graphs:
        o.zero_()
    for g, o, grads in graphs:
        g.replay()
    torch.cuda.synchronize()
    for g, o, grads in graphs:
        assert torch.equal(o, want) and all(torch.equal(a, b) for a, b in zip(grads, wantg))
    fresh = ops.SequencePack([200, 31], [900, 31])
    with pytest.raises(RuntimeError, match="before capturing"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.packed_attention(q, k, v, fresh)
    torch.cuda.synchronize()
    assert torch.equal(ops.packed_attention(q, k, v, fresh), want)


def _with_lse(q, k, v, do, pack):
    o, lse = ops.packed_attention(q, k, v, pack, return_lse=True)
    return o, do, lse
