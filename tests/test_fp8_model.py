"""The 8-bit operators in the framework: the DiT with ``quant: fp8``, the trainer with 8-bit
moments, and the optimizer's checkpoints."""
import copy
import json
import os

import pytest
import torch

from osp_next_b200 import ops
from osp_next_b200.models.lora import inject_lora
from osp_next_b200.models.osp_next import OSPNextModel
from osp_next_b200.parallel.optim import FusedAdamW
from osp_next_b200.quant import FP8Linear, fp8_multi_linear, freeze_fp8_weights

from test_trainer_cpu import _cfg, _main

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(quant, device, dim=256):
    torch.manual_seed(0)
    with torch.device(device):
        return OSPNextModel(dim=dim, ffn_dim=512, num_heads=2, num_layers=2, text_len=16,
                            skiparse_model_type="dual_end", sparse_ratio=2, num_full_blocks=0, quant=quant)


def _inputs(device):
    g = torch.Generator().manual_seed(1)
    return (torch.randn(1, 16, 3, 16, 16, generator=g).to(device), torch.tensor([500.0], device=device),
            torch.randn(1, 16, 4096, generator=g).to(device))


@pytest.mark.parametrize("device", DEVICES)
def test_model_in_fp8_is_near_the_plain_model(device):
    """The same weights: outputs and gradients differ by the quantisation (2^-4 of a value at
    most, some 3 % in the mean of a product), far less than the values themselves."""
    plain, fp8 = _model(None, device), _model("fp8", device)
    fp8.load_state_dict(plain.state_dict())
    assert sum(isinstance(m, FP8Linear) for m in fp8.modules()) == 2 * 10
    for m in (plain, fp8):                       # the head starts at zero in a fresh model
        torch.manual_seed(3)
        torch.nn.init.normal_(m.head.head.weight, std=0.02)
    x, t, ctx = _inputs(device)
    with torch.no_grad():
        a, b = plain(x, t, ctx).float(), fp8(x, t, ctx).float()
        frozen = freeze_fp8_weights(fp8.eval())(x, t, ctx).float()
    assert torch.equal(b, frozen)
    assert ((a - b).norm() / a.norm()).item() < 0.15
    grads = []
    for m in (plain.train(), fp8.train()):
        m(x, t, ctx).float().square().mean().backward()
        grads.append({n: p.grad.float() for n, p in m.named_parameters() if p.grad is not None})
    assert grads[0].keys() == grads[1].keys()
    for n, g in grads[0].items():
        if g.norm() > 1e-6 * max(x.norm() for x in grads[0].values()):
            cos = torch.nn.functional.cosine_similarity(g.flatten(), grads[1][n].flatten(), dim=0).item()
            assert cos > 0.9, (n, cos)


@pytest.mark.parametrize("device", DEVICES)
def test_multi_linear_equals_the_separate_layers(device):
    torch.manual_seed(0)
    layers = [FP8Linear(96, n, device=device) for n in (128, 256, 128)]
    x = torch.randn(2, 5, 96, device=device).to(torch.bfloat16)
    want = torch.cat([m(x) for m in layers], -1)
    assert torch.equal(fp8_multi_linear(x, layers), want)
    with torch.no_grad():
        assert torch.equal(fp8_multi_linear(x, layers), want)
        for m in layers:
            m.freeze_weight()
        assert torch.equal(fp8_multi_linear(x, layers), want)
        layers[1].weight.data.zero_()
        layers[1].freeze_weight()                # a weight frozen anew: the stack is built anew
        new = fp8_multi_linear(x, layers)
    assert torch.equal(new[..., :128], want[..., :128]) and not torch.equal(new, want)
    odd = [FP8Linear(96, n, device=device) for n in (40, 7)]
    assert torch.equal(fp8_multi_linear(x, odd), torch.cat([m(x) for m in odd], -1))


@pytest.mark.parametrize("device", DEVICES)
def test_lora_on_fp8_layers(device):
    """A fresh adapter (B = 0) leaves the fp8 model's output as it was; its factors get gradients."""
    model = _model("fp8", device)
    torch.nn.init.normal_(model.head.head.weight, std=0.02)
    x, t, ctx = _inputs(device)
    with torch.no_grad():
        want = model(x, t, ctx)
    inject_lora(model, 4, 4.0, ["self_attn.q", "self_attn.o", "cross_attn.k", "ffn.0", "ffn.2"])
    with torch.no_grad():
        got = model(x, t, ctx)
    assert ((got - want).float().norm() / want.float().norm()).item() < 2.0 ** -6     # GELU after a bf16 rounding
    model(x, t, ctx).float().square().mean().backward()
    assert all(p.grad is not None for n, p in model.named_parameters() if "lora_" in n)


@pytest.mark.parametrize("device", DEVICES)
def test_optimizer_checkpoints_hold_fp32_moments(device):
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(70, 50), torch.nn.Linear(50, 3)).to(device)
    twin = copy.deepcopy(net)
    x = torch.randn(64, 70, device=device)

    def steps(model, opt, n):
        for _ in range(n):
            model(x).square().mean().backward()
            opt.step()
            opt.zero_grad()
    opt = FusedAdamW(net.parameters(), lr=1e-3, state_bits=8)
    steps(net, opt, 3)
    sd = opt.state_dict()
    for st in sd["state"].values():
        assert set(st) == {"step", "exp_avg", "exp_avg_sq"} and st["exp_avg"].dtype == torch.float32
    # into 8 bits again: the same values (a block whose largest was rounded down may take a smaller scale)
    opt2 = FusedAdamW(twin.parameters(), lr=1e-3, state_bits=8)
    opt2.load_state_dict(copy.deepcopy(sd))
    for a, b in zip(opt.state.values(), opt2.state.values()):
        assert a["step"] == b["step"]
        for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
            assert a[k].shape == b[k].shape and a[k].dtype == b[k].dtype
        assert all(torch.equal(p, q) for p, q in zip(*(ops.adamw8_decode(
            *(s[k] for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"))) for s in (a, b))))
    # into fp32 moments, by either path, and back
    for multi in (False, True):
        opt32 = FusedAdamW(twin.parameters(), lr=1e-3, multi_tensor=multi)
        opt32.load_state_dict(copy.deepcopy(sd))
        steps(twin, opt32, 2)
        opt8 = FusedAdamW(twin.parameters(), lr=1e-3, state_bits=8)
        opt8.load_state_dict(copy.deepcopy(opt32.state_dict()))
        steps(twin, opt8, 1)
    assert all(bool(p.isfinite().all()) for p in twin.parameters())


@pytest.mark.parametrize("device", DEVICES)
def test_optimizer_options(device):
    p = [torch.nn.Parameter(torch.ones(4, device=device))]
    with pytest.raises(ValueError):
        FusedAdamW(p, state_bits=16)
    with pytest.raises(ValueError):
        FusedAdamW(p, state_bits=8, multi_tensor=False)
    # 8-bit, list and per-tensor forms take nearly the same path on a quadratic
    ends = []
    for kw in (dict(), dict(multi_tensor=True), dict(state_bits=8)):
        torch.manual_seed(0)
        w = torch.nn.Parameter(torch.randn(500, device=device))
        skipped = torch.nn.Parameter(torch.ones(3, device=device))
        target = torch.randn(500, device=device)
        opt = FusedAdamW([{"params": [w, skipped]}], lr=0.05, weight_decay=0.0, **kw)
        for _ in range(100):
            opt.zero_grad()
            (w - target).square().sum().backward()
            opt.step()
        assert torch.equal(skipped.detach(), torch.ones_like(skipped))
        ends.append((w.detach() - target).abs().mean().item())
    assert max(ends) < 0.1 and abs(ends[0] - ends[1]) < 1e-4


def test_trainer_with_fp8_and_8bit_moments(tmp_path, monkeypatch):
    import torch.distributed as dist
    for k, v in dict(MASTER_ADDR="127.0.0.1", MASTER_PORT="29633", RANK="0", WORLD_SIZE="1", LOCAL_RANK="0").items():
        monkeypatch.setenv(k, v)
    main, out = _main(), str(tmp_path)
    cfg = _cfg(out, max_steps=2)
    cfg["model_config"]["quant"] = "fp8"
    cfg["optimizer_config"]["state_bits"] = 8
    for _ in range(2):                           # the second run resumes from iteration 2
        main(copy.deepcopy(cfg))
        if dist.is_initialized():
            dist.destroy_process_group()
    recs = [json.loads(line) for line in open(os.path.join(out, "metrics.jsonl"))]
    assert [r["iter"] for r in recs] == [1, 2, 3, 4]
    assert all(r["loss"] == r["loss"] and r["loss"] < 100 for r in recs)


def _fsdp_worker(rank, world, port, out_dir):
    import torch.distributed as dist
    from torch.distributed.checkpoint.state_dict import (StateDictOptions, get_optimizer_state_dict,
                                                         set_optimizer_state_dict)
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.fsdp import fully_shard
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    opts = StateDictOptions(full_state_dict=True)

    def build():
        torch.manual_seed(0)
        net = torch.nn.Sequential(torch.nn.Linear(70, 51), torch.nn.Linear(51, 3))     # odd rows: uneven shards
        return fully_shard(net, mesh=init_device_mesh("cpu", (world,)))

    def steps(net, opt, first, n):
        for i in range(first, first + n):
            for j, p in enumerate(net.parameters()):
                full = torch.randn(p.shape, generator=torch.Generator().manual_seed(100 * i + j))
                p.grad = torch.distributed.tensor.distribute_tensor(full, p.device_mesh, p.placements)
            opt.step()
    net = build()
    opt = FusedAdamW(net.parameters(), lr=1e-2, state_bits=8)
    steps(net, opt, 0, 3)
    full = get_optimizer_state_dict(net, opt, options=opts)
    opt.zero_grad(set_to_none=True)              # as on resume: no gradients yet
    again = FusedAdamW(net.parameters(), lr=1e-2, state_bits=8)
    set_optimizer_state_dict(net, again, copy.deepcopy(full), options=opts)
    names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
    for a, b in zip(opt.state.values(), again.state.values()):
        assert a["step"] == b["step"]
        assert all(torch.equal(x, y) for x, y in zip(*(ops.adamw8_decode(*(s[k] for k in names)) for s in (a, b))))
    state = {n: {k: v for k, v in st.items()} for n, st in full["state"].items()}
    shapes = {n: tuple(p.shape) for n, p in net.named_parameters()}
    assert all(tuple(st[k].shape) == shapes[n] for n, st in state.items() for k in ("exp_avg", "exp_avg_sq"))
    steps(net, again, 3, 1)
    torch.save({"state": state, "params": [p.full_tensor() for p in net.parameters()]},
               os.path.join(out_dir, f"r{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


def test_8bit_moments_on_sharded_parameters(tmp_path):
    """Two ranks with uneven FSDP shards: the full checkpoint has the moments of the whole tensors,
    those of the shards stepped alone, and loading it gives back the same values."""
    import torch.multiprocessing as mp
    from test_distributed_cpu import _port
    mp.start_processes(_fsdp_worker, args=(2, _port(), str(tmp_path)), nprocs=2, join=True, start_method="spawn")
    outs = [torch.load(tmp_path / f"r{r}.pt") for r in range(2)]
    for a, b in zip(outs[0]["params"], outs[1]["params"]):
        assert torch.equal(a, b) and bool(a.isfinite().all())
    # each rank's shards by themselves (rows dealt as FSDP deals them), put together
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(70, 51), torch.nn.Linear(51, 3))
    parts = []
    for rank in range(2):
        shards = [torch.nn.Parameter(p.detach().chunk(2)[rank].clone()) for p in net.parameters()]
        opt = FusedAdamW(shards, lr=1e-2, state_bits=8)
        for i in range(3):
            for j, (p, full) in enumerate(zip(shards, net.parameters())):
                g = torch.randn(full.shape, generator=torch.Generator().manual_seed(100 * i + j))
                p.grad = g.chunk(2)[rank].contiguous()
            opt.step()
        parts.append([st for st in opt.state_dict()["state"].values()])
    for (n, _), a, b in zip(net.named_parameters(), *parts):
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(outs[0]["state"][n][k], torch.cat([a[k], b[k]])), (n, k)
