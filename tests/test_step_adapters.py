"""Adapters of the batch's requests in the decode step (backbone.LatentDecoder.step)."""
import gc

import pytest
import torch

from wsvd_b200.backbone import Adapters, BackboneSpec, LatentDecoder

SPEC = BackboneSpec(layers=2, hidden=512, heads=4, head_dim=128, ffn=1024, rank_k=64, rank_v=64)
WIDTHS = {"qkv": (512, 4 * (128 + 64 + 64)), "o": (512, 512), "up_gate": (512, 2048), "down": (1024, 512)}


def _layers(count, rank, names, device):
    g = torch.Generator().manual_seed(7)
    return [{n: ((torch.randn(count, WIDTHS[n][0], rank, generator=g) / WIDTHS[n][0] ** 0.5).half().to(device),
                 (torch.randn(count, rank, WIDTHS[n][1], generator=g) * 0.2 / rank ** 0.5).half().to(device)) for n in names}
            for _ in range(SPEC.layers)]


def _model(device="cuda"):
    return LatentDecoder(SPEC, batch=3, context=100, capacity=110, device=device, seed=5)


def test_refusals():
    model = _model("cpu")
    x = torch.zeros(3, 512, dtype=torch.float16)
    index = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="one dict per layer"):
        model.step(x, Adapters(index, [{}]))
    with pytest.raises(ValueError, match="unknown projections"):
        model.step(x, Adapters(index, [{}, {"gate": None}]))
    model.fused_elementwise = False
    with pytest.raises(ValueError, match="fused_elementwise"):
        model.step(x, Adapters(index, [{}, {}]))


@pytest.mark.gpu
def test_a_mixed_batch_gives_each_request_what_it_gets_alone_with_its_adapter():
    x = (torch.randn(3, 512, generator=torch.Generator().manual_seed(2)) * 0.5).half().cuda()
    layers = _layers(2, 16, list(WIDTHS), "cuda")
    scale = torch.tensor([0.7, 1.5], device="cuda")

    def step(index):
        return _model().step(x, Adapters(torch.tensor(index, dtype=torch.int32).cuda(), layers, scale))

    mixed = step([1, -1, 0])
    plain = _model().step(x)
    assert torch.equal(mixed[1], plain[1])
    assert torch.equal(mixed[0], step([1, 1, 1])[0]) and torch.equal(mixed[2], step([0, 0, 0])[2])
    assert not torch.equal(mixed[0], plain[0]) and not torch.equal(mixed[2], plain[2])


@pytest.mark.gpu
def test_an_adapter_is_its_product_added_to_the_weights():
    x = (torch.randn(3, 512, generator=torch.Generator().manual_seed(3)) * 0.5).half().cuda()
    layers = _layers(1, 8, list(WIDTHS), "cuda")
    got = _model().step(x, Adapters(torch.zeros(3, dtype=torch.int32).cuda(), layers))
    merged = _model()
    for L, names in zip(merged.layers, layers):
        for name, W in (("qkv", L.Wqkv), ("o", L.Wo), ("up_gate", L.Wug), ("down", L.Wdown)):
            a, b = names[name]
            W.copy_((W.float() + a[0].float() @ b[0].float()).half())
    want = merged.step(x)
    err, size = (got.float() - want.float()).abs().max().item(), want.float().abs().max().item()
    # f16 roundings of the weights against those of the adapters' share, and a latent that rounds the other way now and then
    assert err <= 3e-2 * size, (err, size)


@pytest.mark.gpu
def test_a_captured_step_with_adapters_replays_like_the_eager_one():
    x = (torch.randn(3, 512, generator=torch.Generator().manual_seed(4)) * 0.5).half().cuda()
    ad = Adapters(torch.tensor([0, 1, -1], dtype=torch.int32).cuda(), _layers(2, 16, ["qkv", "down"], "cuda"))
    eager, model = _model(), _model()
    graph, out = model.capture(x, ad)  # (its warm-up is one step)
    eager.step(x, ad)
    eager.advance()
    want = eager.step(x, ad)
    graph.replay()
    torch.cuda.synchronize()
    err = (out.float() - want.float()).abs().max().item()
    assert err <= 2e-2 * want.float().abs().max().item()  # (another split plan: the graph's is made for the capacity)


@pytest.mark.gpu
def test_a_captured_step_keeps_what_it_reads():
    """Input and adapters made inline: nothing else holds them when the graph is replayed and their memory is asked for again."""
    start = (torch.randn(3, 512, generator=torch.Generator().manual_seed(6)) * 0.5).half().cuda()

    def adapters():
        return Adapters(torch.tensor([0, 1, -1], dtype=torch.int32).cuda(), _layers(2, 16, list(WIDTHS), "cuda"),
                        torch.tensor([0.5, 2.0]).cuda())

    held = adapters()
    model = _model()
    graph, want = model.capture(start, held)
    graph.replay()
    want = want.clone()

    model = _model()
    mine = adapters()
    graph, got = model.capture(start.clone(), mine)
    mine.layers[0]["qkv"] = None  # the container is the caller's; the graph keeps the tensors
    del model, mine
    gc.collect()
    sizes = [t.shape for names in held.layers for pair in names.values() for t in pair] + [start.shape]
    junk = [torch.full(s, float("nan"), dtype=torch.float16, device="cuda") for s in sizes * 3]
    ints = [torch.full((3,), 1, dtype=torch.int32, device="cuda") for _ in range(8)]
    floats = [torch.full((2,), float("nan"), device="cuda") for _ in range(8)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    del junk, ints, floats
