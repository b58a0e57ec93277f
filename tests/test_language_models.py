"""The umT5 encoder and the reward backbone on the packed kernels: packed against padded, kernels
against the library path, with the same weights."""
import pytest
import torch

from osp_next_b200 import ops
from osp_next_b200.models import t5
from osp_next_b200.rewards import videoalign as va
from test_videoalign import _tiny_vl

gpu = pytest.mark.gpu
T5 = dict(vocab=100, dim=64, dim_attn=64, dim_ffn=136, num_heads=4, num_layers=2, num_buckets=32, dropout=0.0)


def _t5(shared, **kw):
    torch.manual_seed(0)
    return t5.T5Encoder(**{**T5, "shared_pos": shared, **kw}).eval()


def _prompts(lengths, width):
    ids = torch.randint(1, 100, (len(lengths), width), generator=torch.Generator().manual_seed(3))
    mask = (torch.arange(width)[None] < torch.tensor(lengths)[:, None]).long()
    return ids, mask


@pytest.mark.parametrize("shared", [True, False])
def test_t5_packed_matches_padded(shared):
    enc = _t5(shared)
    lengths = [20, 1, 7, 0]
    ids, mask = _prompts(lengths, 20)
    with torch.no_grad():
        want = enc(ids, mask)
        got = enc(ids[mask > 0], pack=ops.SequencePack(lengths, device="cpu"))
    assert torch.allclose(got, want[mask > 0], atol=1e-5)


def test_t5_bias_table_is_the_bias():
    e = t5.T5RelativeEmbedding(32, 4, True)
    full, table = e(300, 300)[0], e.table(300)
    i = torch.arange(300)
    assert torch.equal(table[:, (i[None] - i[:, None]) + 299], full)


def test_t5_encoder_model_on_the_cpu_is_unchanged():
    enc = t5.T5EncoderModel(text_len=24, dtype=torch.float32, device="cpu", encoder=_t5(False))
    ids, mask = _prompts([20, 3], 20)
    out = enc(ids, mask)
    with torch.no_grad():
        want = enc.model(ids, mask)
    assert out.shape == (2, 24, 64) and torch.equal(out[0, :20], want[0]) and torch.equal(out[1, :3], want[1, :3])
    assert (out[1, 3:] == 0).all() and (out[0, 20:] == 0).all()


@pytest.mark.parametrize("side", ["right", "left", "none", "holes"])
def test_reward_backbone_with_kernels_matches_library(side):
    ids = torch.randint(3, 280, (3, 24), generator=torch.Generator().manual_seed(1))
    mask = torch.ones_like(ids)
    if side == "right":
        mask[1, 15:], mask[2, 1:] = 0, 0
    elif side == "left":
        mask[1, :9] = 0
    elif side == "holes":
        mask[1, 5:9] = 0
    ids[:, 10], ids[:, 12], ids[:, 14] = 295, 296, 297
    ids[2, 0] = 295
    model = va.VideoAlignRewardModel(_tiny_vl(), output_dim=3, special_token_ids=[295, 296, 297])
    with torch.no_grad():
        h0 = model._hidden(ids, mask)
        model.use_kernels().use_kernels()
        h1 = model._hidden(ids, mask)
        assert torch.allclose(h0[mask > 0], h1[mask > 0], atol=1e-5)
        assert torch.isfinite(h1).all()
        if side == "none":
            assert torch.allclose(model._hidden(ids, None)[mask > 0], h1[mask > 0], atol=1e-6)
    assert model.vl.config.text_config._attn_implementation == va.ATTENTION_NAME
    assert model.vl.config.vision_config._attn_implementation != va.ATTENTION_NAME


def test_reward_backbone_gradients_with_kernels():
    ids = torch.randint(3, 280, (2, 12), generator=torch.Generator().manual_seed(1))
    mask = torch.ones_like(ids)
    mask[1, 7:] = 0
    grads = []
    for kernels in (False, True):
        model = va.VideoAlignRewardModel(_tiny_vl(), output_dim=1, reward_token="last")
        if kernels:
            model.use_kernels()
        h = model._hidden(ids, mask)[mask > 0]
        h.square().sum().backward()
        grads.append({n: p.grad for n, p in model.named_parameters() if p.grad is not None})
    assert grads[0].keys() == grads[1].keys()
    for n, g in grads[0].items():
        assert torch.allclose(g, grads[1][n], atol=1e-4 * max(1.0, float(g.abs().max()))), n


# ---------------------------------------------------------------------------- GPU

@gpu
@pytest.mark.parametrize("shared", [True, False])
def test_gpu_t5_encoder_model(shared):
    """bf16 on the kernels, packed, against the same bf16 weights in fp32 on the CPU.  Each of two
    layers rounds some ten values on a path to bf16, errors of half a step each: 2 x 10 x 2^-8 of the
    values' size if none cancelled, a quarter of it in the norm is far above what random ones give."""
    enc = _t5(shared).to(torch.bfloat16)
    plain = _t5(shared)
    plain.load_state_dict({k: v.float() for k, v in enc.state_dict().items()})
    ids, mask = _prompts([20, 1, 33, 0], 40)
    with torch.no_grad():
        want = plain(ids, mask)
    model = t5.T5EncoderModel(text_len=48, dtype=torch.bfloat16, device="cuda", encoder=enc)
    n0 = ops._ext.launch_count()
    out = model(ids, mask)
    assert ops._ext.launch_count() - n0 == 2 * 2          # attention and the feed-forward block, two layers
    assert out.shape == (4, 48, 64) and out.dtype == torch.bfloat16
    real = torch.zeros(4, 48, dtype=torch.bool)
    real[:, :40] = mask > 0
    assert (out.cpu()[~real] == 0).all()
    d = out.cpu().float()[real] - want[mask > 0]
    assert d.norm() <= 2 * 10 * 2.0 ** -8 / 4 * want[mask > 0].norm()
    holes = mask.clone()
    holes[0, 4] = 0                                       # not a prefix: the padded path
    with torch.no_grad():
        ctx = model.model(ids.cuda(), holes.cuda())
    assert torch.equal(model(ids, holes)[0, :19], ctx[0, :19])
    with pytest.raises(ValueError, match="text_len"):
        t5.T5EncoderModel(text_len=8, dtype=torch.bfloat16, device="cuda", encoder=enc)(ids, mask)


@gpu
def test_gpu_reward_backbone():
    """As above: two layers, bf16 kernels against fp32 on the CPU."""
    ids = torch.randint(3, 280, (3, 40), generator=torch.Generator().manual_seed(1))
    mask = torch.ones_like(ids)
    mask[1, 15:], mask[2, 1:] = 0, 0
    model = va.VideoAlignRewardModel(_tiny_vl(), output_dim=3, reward_token="last")
    model.bfloat16()
    state = {k: v.float() for k, v in model.state_dict().items()}
    plain = va.VideoAlignRewardModel(_tiny_vl(), output_dim=3, reward_token="last")
    plain.load_state_dict(state)
    with torch.no_grad():
        want = plain._hidden(ids, mask)[mask > 0]
        model.cuda().use_kernels()
        n0 = ops._ext.launch_count()
        got = model._hidden(ids.cuda(), mask.cuda()).cpu()
    assert ops._ext.launch_count() - n0 == 2 * 2
    assert torch.isfinite(got).all()
    assert (got.float()[mask > 0] - want).norm() <= 2 * 10 * 2.0 ** -8 / 4 * want.norm()


@gpu
def test_gpu_rope_of_heads_without_norm():
    """The DiT's attention without q/k norm rotates on the kernel, forward and backward."""
    from osp_next_b200.models import functional as Fn
    from osp_next_b200.ops import reference as ref
    pos = torch.randint(0, 60, (50, 3), device="cuda")
    freqs = ref.rope_freqs(64).cuda()
    x = torch.randn(2, 50, 3, 64, device="cuda", requires_grad=True)
    do = torch.randn(2, 50, 3, 64, device="cuda")
    n0 = ops._ext.launch_count()
    y = Fn.apply_rope(x, pos, freqs)
    g, = torch.autograd.grad(y, x, do)
    assert ops._ext.launch_count() - n0 == 2
    want = ref.apply_rope(x, pos, freqs)
    gw, = torch.autograd.grad(want, x, do)
    # angles to 60 in fp32 on one side: half a step of 2^-18 each
    assert torch.allclose(y, want, atol=5e-5) and torch.allclose(g, gw, atol=5e-5)
