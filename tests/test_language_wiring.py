"""Calls around the umT5 encoder and the reward backbone that reach their kernels by another way than the
scorer and the prompt encoder: the backbone called directly, recomputed in the backward pass, generating;
layers replaced, wrapped or watched after the model was made."""
import threading

import pytest
import torch

from osp_next_b200 import ops
from osp_next_b200.models import t5
from osp_next_b200.rewards import videoalign as va
from test_videoalign import _tiny_vl

gpu = pytest.mark.gpu


def _batch(side, B=3, L=24, seed=1):
    ids = torch.randint(3, 280, (B, L), generator=torch.Generator().manual_seed(seed))
    mask = torch.ones_like(ids)
    if side == "right":
        mask[1, 15:], mask[2, 1:] = 0, 0
    elif side == "left":
        mask[1, :9], mask[2, :L - 1] = 0, 0
    elif side == "holes":
        mask[1, 5:9] = 0
    return ids, mask


def _backbones():
    """The same random backbone without and with the kernels."""
    return _tiny_vl(), va.VideoAlignRewardModel(_tiny_vl(), output_dim=1, reward_token="last").use_kernels().vl


@pytest.mark.parametrize("side", ["right", "left", "none", "holes"])
def test_backbone_called_directly_keeps_its_mask(side):
    ids, mask = _batch(side)
    plain, kernels = _backbones()
    with torch.no_grad():
        want, got = (m.model(input_ids=ids, attention_mask=mask).last_hidden_state for m in (plain, kernels))
    assert torch.allclose(got[mask > 0], want[mask > 0], atol=1e-5)


@pytest.mark.parametrize("side", ["right", "left", "holes"])
@pytest.mark.parametrize("reentrant", [True, False])
def test_backbone_recomputed_in_the_backward_pass(side, reentrant):
    ids, mask = _batch(side)
    grads = []
    for m, recompute in zip(_backbones(), (False, True)):
        if recompute:
            m.gradient_checkpointing_enable({"use_reentrant": reentrant})
            m.train()
        x = m.get_input_embeddings()(ids).detach().requires_grad_(True)
        h = m.model(inputs_embeds=x, attention_mask=mask, use_cache=False,
                    position_ids=torch.arange(ids.shape[1]).expand(3, *ids.shape)).last_hidden_state
        h[mask > 0].square().sum().backward()
        grads.append({"x": x.grad, **{n: p.grad for n, p in m.named_parameters() if p.grad is not None}})
    assert "x" in grads[1]
    for n, g in grads[1].items():
        want = grads[0][n]
        assert torch.allclose(g, want, atol=1e-4 * max(1.0, float(want.abs().max()))), n


@pytest.mark.parametrize("side", ["left", "none"])
def test_backbone_generates(side):
    """A prompt at once, then single tokens over a cache."""
    ids, mask = _batch(side)
    plain, kernels = _backbones()
    want, got = (m.generate(input_ids=ids, attention_mask=mask, max_new_tokens=4, do_sample=False, pad_token_id=0)
                 for m in (plain, kernels))
    assert torch.equal(got, want)


def test_backbone_with_a_mask_of_its_callers():
    """A mask [B, 1, L, L] made by the caller."""
    ids, _ = _batch("none")
    m4 = torch.ones(24, 24, dtype=torch.bool).tril().triu(-5)[None, None].expand(3, 1, 24, 24)
    with torch.no_grad():
        want, got = (m.model(input_ids=ids, attention_mask=m4).last_hidden_state for m in _backbones())
    assert torch.allclose(got, want, atol=1e-5)


def test_backbone_config_stays_during_a_call():
    """Batches with holes in their masks in one thread, others in a second one, on the same model."""
    model = va.VideoAlignRewardModel(_tiny_vl(), output_dim=1, reward_token="last")
    batches = [_batch("holes"), _batch("left", seed=2)]
    with torch.no_grad():
        want = [model._hidden(*b) for b in batches]
    model.use_kernels()

    def refuse(*a, **k):
        raise AssertionError("the shared configuration is switched during a call")
    model.vl.set_attn_implementation = refuse
    got = [[], []]

    def work(i):
        with torch.no_grad():
            for _ in range(5):
                got[i].append(model._hidden(*batches[i]))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i, (_, mask) in enumerate(batches):
        assert len(got[i]) == 5
        for h in got[i]:
            assert torch.allclose(h[mask > 0], want[i][mask > 0], atol=1e-5)


def test_backbone_in_training_drops_attention_weights(monkeypatch):
    """attention_dropout of a backbone in training: every weight dropped leaves the layers without attention."""
    ids, mask = _batch("left")
    plain, kernels = _backbones()
    out = []
    for m in (plain, kernels):
        m.train()
        for layer in m.model.language_model.layers:
            layer.self_attn.attention_dropout = 1.0
        with torch.no_grad():
            out.append(m.model(input_ids=ids, attention_mask=mask).last_hidden_state)
    assert torch.allclose(out[0], out[1], atol=1e-5)


def _touch(block, names, how):
    """Adapters, quantisation, hooks or another forward on the layers ``names`` of a gated block."""
    torch.manual_seed(5)
    if how == "lora":
        from osp_next_b200.models.lora import LoraLinear, inject_lora
        assert len(inject_lora(block, 8, 16.0, names)) == len(names)
        for m in block.modules():
            if isinstance(m, LoraLinear):
                for part in (m.lora_A, m.lora_B):
                    torch.nn.init.normal_(part["default"].weight)
    elif how == "quantised":
        from osp_next_b200.quant.fp8 import FP8Linear
        for n in names:
            old = block.get_submodule(n)
            new = FP8Linear(old.in_features, old.out_features, bias=False)
            new.weight = old.weight
            parent, _, leaf = n.rpartition(".")
            setattr(block.get_submodule(parent), leaf, new)
    elif how == "bias":
        for n in names:
            m = block.get_submodule(n)
            m.bias = torch.nn.Parameter(torch.randn(m.out_features, dtype=m.weight.dtype, device=m.weight.device))
    elif how == "forward":
        m = block.get_submodule(names[0])
        plain = m.forward
        m.forward = lambda x: 2 * plain(x)
    else:
        hook = {"hook": "register_forward_hook", "pre": "register_forward_pre_hook",
                "backward": "register_full_backward_hook"}[how]
        getattr(block.get_submodule(names[-1]), hook)(
            {"hook": lambda m, a, y: 2 * y, "pre": lambda m, a: (2 * a[0],), "backward": lambda m, a, g: None}[how])


TOUCHES = ["lora", "quantised", "bias", "forward", "hook", "pre", "backward"]


def test_t5_feed_forward_knows_its_layers():
    names = ["gate.0", "fc1", "fc2"]
    ffn = t5.T5FeedForward(16, 40, 0.0)
    assert ffn._plain()
    for how in TOUCHES:
        ffn = t5.T5FeedForward(16, 40, 0.0)
        _touch(ffn, names, how)
        assert not ffn._plain(), how
    ffn = t5.T5FeedForward(16, 40, 0.0)
    ffn.gate[1] = torch.nn.GELU()
    assert not ffn._plain()
    ffn = t5.T5FeedForward(16, 40, 0.0)
    ffn.gate.register_forward_hook(lambda m, a, y: 2 * y)
    assert not ffn._plain()


@gpu
@pytest.mark.parametrize("how", TOUCHES)
def test_gpu_t5_feed_forward_runs_its_layers(how):
    """The module gives what its layers give one after another, whatever they are."""
    torch.manual_seed(0)
    ffn = t5.T5FeedForward(64, 136, 0.0).eval().to("cuda", torch.bfloat16)
    x = torch.randn(5, 64, device="cuda").bfloat16()
    with torch.no_grad():
        before = ffn(x)
        _touch(ffn, ["gate.0", "fc1", "fc2"], how)
        want = ffn.cuda().fc2(ffn.fc1(x) * ffn.gate(x))
        got = ffn(x)
    assert torch.equal(got, want)
    assert how == "backward" or not torch.equal(got, before)


@pytest.mark.parametrize("how", TOUCHES)
def test_backbone_mlp_runs_its_layers(how):
    """Layers replaced, wrapped or watched after use_kernels."""
    torch.manual_seed(0)
    plain, kernels = (m.model.language_model.layers[0].mlp for m in _backbones())
    x = torch.randn(5, 64)
    with torch.no_grad():
        before = kernels(x)
        assert torch.allclose(before, plain(x), atol=1e-5)
        for m in (plain, kernels):
            _touch(m, ["gate_proj", "up_proj", "down_proj"], how)
        want, got = plain(x), kernels(x)
    assert torch.equal(got, want)
    assert how == "backward" or not torch.equal(got, before)


@gpu
def test_gpu_backbone_in_other_types_and_heads():
    """fp32, and heads that the packed kernel does not take: the library's attention.  fp32 sums of some 200
    terms a layer on both sides, 2^-24 each."""
    ids, mask = _batch("left")
    with torch.no_grad():
        want = _tiny_vl().model(input_ids=ids, attention_mask=mask).last_hidden_state
        m = va.VideoAlignRewardModel(_tiny_vl(), output_dim=1, reward_token="last").cuda().use_kernels().vl
        n0 = ops._ext.launch_count()
        got = m.model(input_ids=ids.cuda(), attention_mask=mask.cuda()).last_hidden_state.cpu()
        assert ops._ext.launch_count() == n0
    assert (got - want)[mask > 0].norm() <= 2 * 200 * 2.0 ** -24 * want[mask > 0].norm()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype,dim,grad", [(torch.float32, 64, False), (torch.float32, 64, True), (torch.bfloat16, 64, True),
                                            (torch.float32, 48, False)])
def test_t5_packed_in_other_types_and_under_autograd(device, dtype, dim, grad):
    """Packed prompts in a type, with heads or gradients that the packed kernel does not take: elementary
    operations in the model's type, here against 64 bits.  Bounds: two layers of some ten roundings on a path, half
    a step each, were none to cancel, with sums of some 100 terms in fp32 (2^-24 each) in the place of bf16's
    steps for fp32."""
    cfg = dict(vocab=100, dim=dim, dim_attn=dim, dim_ffn=136, num_heads=4, num_layers=2, num_buckets=32, dropout=0.0,
               shared_pos=True)
    torch.manual_seed(0)
    enc = t5.T5Encoder(**cfg).eval().to(dtype)
    plain = t5.T5Encoder(**cfg).eval()
    plain.load_state_dict({k: v.float() for k, v in enc.state_dict().items()})
    enc, plain = enc.to(device), plain.double().to(device)
    lengths = [20, 1, 33, 0]
    ids = torch.randint(1, 100, (sum(lengths),), generator=torch.Generator().manual_seed(3)).to(device)
    pack = ops.SequencePack(lengths, device=device)
    out = []
    for m in (enc, plain):
        with torch.set_grad_enabled(grad):
            y, at = [], 0
            if m is enc:
                y = m(ids, pack=pack)
            else:
                for n in lengths[:3]:
                    y.append(m(ids[None, at:at + n], torch.ones(1, n, device=device))[0])
                    at += n
                y = torch.cat(y)
            out.append([y.detach().double()])
            if grad:
                # squares would cancel: rows leave a norm with the same sum of them
                (y * torch.linspace(-1, 1, y.numel(), device=device).view(y.shape).to(y.dtype)).sum().backward()
                out[-1] += [p.grad.double() for p in m.parameters()]
    bound = 2 * 10 * (2.0 ** -8 if dtype == torch.bfloat16 else 100 * 2.0 ** -24) * (4 if grad else 1)
    for a, b in zip(*out):
        assert (a - b).norm() <= bound * b.norm()


def _tangents(f, x, t):
    from torch.autograd import forward_ad as fw
    with torch.no_grad(), fw.dual_level():
        return fw.unpack_dual(f(fw.make_dual(x, t))).tangent


@gpu
@pytest.mark.parametrize("how", ["forward_mode", "jvp", "vmap", "double"])
def test_gpu_transforms_of_t5_feed_forward(how):
    """What torch does with the modules one by one it does with the block: derivatives forward, over a batch of
    calls and of derivatives.  bf16: some four roundings a value on either side."""
    torch.manual_seed(0)
    ffn = t5.T5FeedForward(64, 136, 0.0).eval().requires_grad_(False).to("cuda", torch.bfloat16)
    x, t = (torch.randn(5, 64, device="cuda").bfloat16() for _ in range(2))

    def parts(z):
        return ffn.fc2(ffn.fc1(z) * ffn.gate(z))

    def result(f):
        if how == "forward_mode":
            return _tangents(f, x, t)
        if how == "jvp":
            return torch.func.jvp(f, (x,), (t,))[1]
        if how == "vmap":
            return torch.func.vmap(f)(x)
        leaf = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(f(leaf), leaf, t, create_graph=True)
        return torch.autograd.grad(g, leaf, x)[0]
    got, want = result(ffn), result(parts)
    assert got is not None and (got.float() - want.float()).norm() <= 8 * 2.0 ** -8 * want.float().norm()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gpu_apply_rope_is_fp32(dtype):
    """The DiT's rotation gives fp32 whatever x is, on both devices, and takes part in torch's transforms."""
    from osp_next_b200.models import functional as Fn
    from osp_next_b200.ops import reference as ref
    pos, freqs = torch.randint(0, 60, (50, 3), device="cuda"), ref.rope_freqs(64).cuda()
    x, t = (torch.randn(2, 50, 3, 64, device="cuda").to(dtype) for _ in range(2))
    want = ref.apply_rope(x, pos, freqs)
    got = Fn.apply_rope(x, pos, freqs)
    # angles to 60 in fp32 on one side: half a step of 2^-18 each
    assert got.dtype == want.dtype == torch.float32 and torch.allclose(got, want, atol=5e-5)

    def f(z):
        return Fn.apply_rope(z, pos, freqs)
    assert torch.allclose(_tangents(f, x, t), ref.apply_rope(t, pos, freqs), atol=5e-5)
    assert torch.allclose(torch.func.vmap(f)(x[:, None])[:, 0], want, atol=5e-5)


@gpu
def test_gpu_operators_under_transforms():
    """No tangent is dropped by the operators of the language models."""
    from osp_next_b200.models import functional as Fn
    pack, table = ops.SequencePack([3, 17]), ops.rotary_table(16, 20)
    pos = torch.arange(20, device="cuda")
    g = torch.Generator("cuda").manual_seed(1)
    x, t = (torch.randn(20, 2, 16, generator=g, device="cuda") for _ in range(2))
    w = [torch.randn(*s, generator=g, device="cuda") for s in ((40, 16), (40, 16), (16, 40))]
    for f in (lambda z: Fn.rotary(z, None, pos, table)[0], lambda z: Fn.packed_attention(z, z, z, pack),
              lambda z: Fn.gated_ffn(z, *w)):
        got = _tangents(f, x, t)
        assert got is not None and torch.allclose(torch.func.jvp(f, (x,), (t,))[1], got, atol=1e-4)


class _Wrapped(torch.nn.Module):
    """What a caller's shard function or another encoder may be: ids and mask in, [B, L, dim] out."""

    def __init__(self, encoder):
        super().__init__()
        self.module = encoder

    def forward(self, ids, mask):
        return self.module(ids, mask)


def _wraps(device, dtype):
    torch.manual_seed(0)
    cfg = dict(vocab=100, dim=64, dim_attn=64, dim_ffn=136, num_heads=4, num_layers=1, num_buckets=32, dropout=0.0)
    enc = t5.T5Encoder(**cfg)
    ids = torch.randint(1, 100, (2, 20), generator=torch.Generator().manual_seed(3))
    mask = (torch.arange(20)[None] < torch.tensor([20, 3])[:, None]).long()
    out = [t5.T5EncoderModel(text_len=24, dtype=dtype, device=device, encoder=enc, shard_fn=f)
           for f in (None, lambda m: _Wrapped(m).to(device, dtype))]
    assert not out[1]._packs()
    return [m(ids, mask).float() for m in out]


def test_prompt_encoder_with_a_wrapped_encoder():
    a, b = _wraps("cpu", torch.float32)
    assert torch.allclose(a, b, atol=1e-6)


@gpu
def test_gpu_prompt_encoder_with_a_wrapped_encoder():
    """Packed and padded: one layer of some ten roundings to bf16, none cancelled."""
    a, b = _wraps("cuda", torch.bfloat16)
    assert (a - b).norm() <= 10 * 2.0 ** -8 * b.norm()


def test_kernels_fit_the_backbones_that_have_their_layers():
    import types
    vl = _tiny_vl()
    assert va._kernels_fit(vl)
    text = vl.config.text_config
    for other in (types.SimpleNamespace(config=vl.config),                                  # no text layers found
                  types.SimpleNamespace(config=vl.config, model=types.SimpleNamespace()),
                  types.SimpleNamespace(config=text, model=vl.model),                       # no text config
                  types.SimpleNamespace(config=types.SimpleNamespace(), model=vl.model)):
        assert not va._kernels_fit(other)
    text.use_sliding_window = True
    assert not va._kernels_fit(vl)
    text.use_sliding_window, text.head_dim = False, 12
    assert not va._kernels_fit(vl)


@gpu
@pytest.mark.parametrize("side", ["left", "holes"])
@pytest.mark.parametrize("reentrant", [True, False])
def test_gpu_backbone_recomputed_in_the_backward_pass(side, reentrant):
    """The same gradients with and without recomputation: kernels and library repeat themselves."""
    ids, mask = (t.cuda() for t in _batch(side))
    grads = []
    for recompute in (False, True):
        m = va.VideoAlignRewardModel(_tiny_vl().bfloat16(), output_dim=1, reward_token="last").cuda().use_kernels().vl
        if recompute:
            m.gradient_checkpointing_enable({"use_reentrant": reentrant})
            m.train()
        x = m.get_input_embeddings()(ids).detach().requires_grad_(True)
        h = m.model(inputs_embeds=x, attention_mask=mask, use_cache=False,
                    position_ids=torch.arange(ids.shape[1], device="cuda").expand(3, *ids.shape)).last_hidden_state
        (h[mask > 0] * torch.linspace(-1, 1, 64, device="cuda").bfloat16()).sum().backward()
        grads.append([x.grad, *(p.grad for p in m.parameters() if p.grad is not None)])
    assert len(grads[0]) == len(grads[1]) and torch.isfinite(grads[0][0]).all() and grads[0][0].any()
    for a, b in zip(*grads):
        assert torch.equal(a, b)
    ops.check_device_errors()


@gpu
@pytest.mark.parametrize("how", ["global_hook", "compiled", "fake", "autocast"])
def test_gpu_t5_feed_forward_as_its_layers_would(how):
    """Hooks on every module, tracing, tensors without data, and autocast to another type: what the layers do one
    after another."""
    torch.manual_seed(0)
    ffn = t5.T5FeedForward(64, 136, 0.0).eval().requires_grad_(False).to("cuda", torch.bfloat16)
    x = torch.randn(5, 64, device="cuda").bfloat16()
    want = ffn.fc2(ffn.fc1(x) * ffn.gate(x))
    if how == "global_hook":
        seen = []
        hook = torch.nn.modules.module.register_module_forward_hook(lambda m, a, y: seen.append(m))
        try:
            assert torch.equal(ffn(x), want)
        finally:
            hook.remove()
        assert all(any(m is s for s in seen) for m in (ffn.gate[0], ffn.fc1, ffn.fc2))
    elif how == "compiled":
        assert torch.equal(torch.compile(ffn, backend="eager", fullgraph=True)(x), want)
    elif how == "fake":
        from torch._subclasses.fake_tensor import FakeTensorMode
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            y = ffn(mode.from_tensor(x))
        assert y.shape == want.shape and y.dtype == want.dtype and y.device.type == "cuda"
    else:
        with torch.autocast("cuda", torch.float16):
            got, want = ffn(x), ffn.fc2(ffn.fc1(x) * ffn.gate(x))
        assert got.dtype == want.dtype == torch.float16 and torch.equal(got, want)
        with torch.autocast("cuda", torch.bfloat16):
            assert ffn(x).dtype == torch.bfloat16


@gpu
@pytest.mark.parametrize("dim", [96, 288])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gpu_apply_rope_qk(dtype, dim):
    """One launch for q and k in bf16, and the same bf16 values as from fp32; heads of any size."""
    from osp_next_b200.models import functional as Fn
    from osp_next_b200.ops import reference as ref
    pos, freqs = torch.randint(0, 60, (50, 3), device="cuda"), ref.rope_freqs(dim).cuda()
    q, k = (torch.randn(2, 50, 3, dim, device="cuda").to(dtype) for _ in range(2))
    n0 = ops._ext.launch_count()
    got = Fn.apply_rope_qk(q, k, pos, freqs)
    launches = ops._ext.launch_count() - n0
    assert launches == (0 if dim > 256 else 1 if dtype == torch.bfloat16 else 2)
    for g, x in zip(got, (q, k)):
        one = Fn.apply_rope(x, pos, freqs)
        assert one.dtype == torch.float32 and torch.equal(g.bfloat16(), one.bfloat16())
        # angles to 60 in fp32 on one side: half a step of 2^-18 each
        assert torch.allclose(one, ref.apply_rope(x, pos, freqs), atol=1e-4)
    ops.check_device_errors()
