"""Microscaled formats on the device: calls that earlier tests leave out.

The forward of a quantised model between writes of every kind and replays, and the projection's paths that only large batches, rows
already in codes or very wide rows take.  Bounds as in the tests of the operators: a sum of K exact products in float32 is within
K 2^-23 of the sum of the magnitudes, the bias adds one addition, the type half a step."""
import pytest
import torch

import crosslayer_coding_amd as cca
from crosslayer_coding_amd import synth
from oracle import mx_oracle as orc

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


# ---- a model whose encoder is quantised ----------------------------------------------------------------------------

def _model(dev, T=40, dtype="bfloat16", fn="batchtopk", d=256, F=1024, L=3):
    model, inputs, x = synth.build_model(synth.Workload("mx", 9, L, d, F, T, dtype, fn, 16, "per_layer", "none"), dev)
    return model, inputs, x


def _true(model, inputs, x):
    """The pre-activations are those of the weights as they are now."""
    w = torch.stack([e.weight.detach() for e in model.encoder_module.encoders]).cpu()
    b = torch.stack([e.bias_param.detach() for e in model.encoder_module.encoders]).cpu().double().unsqueeze(1)
    xq, wq = orc.round_trip(x.cpu(), "mxfp4"), orc.round_trip(w, "mxfp4")
    want = xq @ wq.transpose(1, 2) + b
    tol = (xq.abs() @ wq.abs().transpose(1, 2) + b.abs()) * (w.shape[-1] + 1) * 2.0 ** -23 + want.abs() * torch.finfo(model.dtype).eps / 2 * 1.01 + 1e-30
    pre, _ = model._encode_all_layers(inputs)
    for l in inputs:
        assert bool(((pre[l].cpu().double() - want[l]).abs() <= tol[l]).all()), l


def _capture(model, inputs):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            model(inputs)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = model(inputs)
    return g, out


@pytest.mark.parametrize("how", ["mul_", "load_state_dict"])
def test_a_captured_forward_lives_through_writes_that_the_host_sees(dev, how):
    """Capture, write, an eager forward on another stream, other tensors in the memory that is free now, replay."""
    model, inputs, x = _model(dev)
    model.quantise_encoder()
    with torch.no_grad():
        g, out = _capture(model, inputs)
        at = [t.data_ptr() for t in model.encoder_module._mx_state]
        for trial in range(3):
            if how == "mul_":
                model.encoder_module.encoders[trial].weight.mul_(-1.5)
            else:
                model.load_state_dict({k: v * 0.75 for k, v in model.state_dict().items()})
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                model(inputs)
                others = [torch.full((n,), 7, dtype=torch.int32, device=dev) for n in (3, 48, 96, 128) for _ in range(8)]
            torch.cuda.current_stream().wait_stream(s)
            others += [torch.full((n,), 7, dtype=torch.int32, device=dev) for n in (3, 48, 96, 128) for _ in range(8)]
            assert at == [t.data_ptr() for t in model.encoder_module._mx_state]
            if trial == 2:
                model.encoder_module.encoders[0].weight.data.neg_()         # seen by the replay alone
            g.replay()
            torch.cuda.synchronize()
            got = {l: v.clone() for l, v in out.items()}
            assert all(bool((t == 7).all()) for t in others)
            want = model(inputs)
            assert all(torch.equal(got[l], want[l]) for l in got), trial
            _true(model, inputs, x)


def test_a_write_while_nobody_watched_is_seen_when_somebody_does_again(dev):
    model, inputs, x = _model(dev)
    enc = model.encoder_module
    with torch.no_grad():
        enc.watch_parameter_data = False
        model.quantise_encoder()
        enc.encoders[1].weight.mul_(-1.5)
        _true(model, inputs, x)
        for lin in enc.encoders:
            lin.weight.data.mul_(0.5)
        enc.watch_parameter_data = True
        model.get_preactivations(inputs[2], 2)
        _true(model, inputs, x)


def test_a_replay_that_makes_the_copy_takes_its_fingerprints_too(dev):
    """Weights put in for one replay and taken out again, past the version counters; the graph was captured right after a write."""
    model, inputs, x = _model(dev)
    model.quantise_encoder()
    weight = model.encoder_module.encoders[1].weight
    with torch.no_grad():
        model(inputs)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            model(inputs)
        torch.cuda.current_stream().wait_stream(s)
        weight.mul_(-0.5)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = model(inputs)
        for trial in range(3):
            want = {l: v.clone() for l, v in model(inputs).items()}
            kept = weight.detach().clone()
            weight.data.mul_(0.3)
            g.replay()
            torch.cuda.synchronize()
            got = {l: v.clone() for l, v in out.items()}
            other = model(inputs)
            assert all(torch.equal(got[l], other[l]) for l in got)
            g.replay()
            weight.data.copy_(kept)
            again = model(inputs)
            assert all(torch.equal(again[l], want[l]) for l in want), trial
            _true(model, inputs, x)


def test_a_copy_that_is_first_made_under_a_capture(dev):
    model, inputs, x = _model(dev)
    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            model(inputs)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            model.quantise_encoder()
            out = model(inputs)
        want = {l: v.clone() for l, v in model(inputs).items()}
        _true(model, inputs, x)
        for trial in range(3):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(out[l], want[l]) for l in want), trial
            again = model(inputs)
            assert all(torch.equal(again[l], want[l]) for l in want), trial
        model.encoder_module.encoders[0].weight.data.neg_()
        _true(model, inputs, x)


# ---- the projection's paths ----------------------------------------------------------------------------------------

def _whole_numbers(shape, top, seed):
    """Small whole numbers, one element of each block fixed so that every block's scale is 1, times a scale per block."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randint(-3, 4, shape, generator=g).float()
    v[..., top::32] = 4.0
    blocks = torch.tensor([1.0, 2.0, 0.5, 8.0])[torch.randint(0, 4, (*shape[:-1], -(-shape[-1] // 32)), generator=g)]
    return v * blocks.repeat_interleave(32, dim=-1)[..., :shape[-1]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("F", [4096, 4100])
@pytest.mark.parametrize("d", [512, 640, 768, 1024, 2048])
def test_project_of_several_tiles_a_workgroup(dev, dtype, F, d):
    """576 and 612 tiles of 2 to 8 stages: a workgroup takes a second and a third one, whose stages follow each other while the tile
    before leaves.  Every partial sum is a multiple of 1/4 below 2^22, so sums are exact in any order and the results are theirs,
    rounded once.  F = 4096: rows of whole cache lines."""
    L, T = 4, 2100
    w = cca.mx.quantise(_whole_numbers((L, F, d), 1, 1).to(dev))
    b = (torch.arange(L * F).reshape(L, F) % 200 - 100).to(dtype).to(dev)
    w64 = w.dequantise().double()
    for trial in range(2):
        x = _whole_numbers((L, T, d), 0, 2 + trial).to(dtype).to(dev)
        out = torch.full((L, T, F), float("nan"), dtype=dtype, device=dev)
        cca.mx.project(x, w, b, out=out)
        for l in range(L):
            want = torch.mm(x[l].double(), w64[l].t().contiguous()) + b[l].double()
            assert torch.equal(out[l], want.to(dtype)), (trial, l)
    for _ in range(3):
        assert torch.equal(cca.mx.project(x, w, b), out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,T,F,d", [(2, 300, 520, 640), (1, 512, 512, 512), (2, 256, 300, 768), (3, 70, 1000, 96), (1, 1000, 260, 2048), (4, 2100, 4096, 768)])
def test_project_of_rows_in_codes_by_tiles(dev, dtype, L, T, F, d):
    """Rows that come in codes, whole tiles of whole stages and others, give what the same rows quantised on the way in give."""
    g = torch.Generator().manual_seed(T + d)
    x = torch.randn(L, T, d, generator=g).to(dtype).to(dev)
    w = cca.mx.quantise((torch.randn(L, F, d, generator=g) / d ** 0.5).to(dev))
    b = torch.randn(L, F, generator=g).to(dtype).to(dev)
    xq = cca.mx.quantise(x)
    out = torch.full((L, T, F), float("nan"), dtype=dtype, device=dev)
    cca.mx.project(xq, w, b, out=out)
    assert torch.equal(out, cca.mx.project(x, w, b))
    x64, w64 = xq.dequantise().double(), w.dequantise().double()
    for l in range(L):
        want = torch.mm(x64[l], w64[l].t().contiguous()) + b[l].double()
        mag = torch.mm(x64[l].abs(), w64[l].abs().t().contiguous()) + b[l].double().abs()
        tol = mag * (d + 1) * 2.0 ** -23 + want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert bool(((out[l].double() - want).abs() <= tol).all()), l


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,T,F,d", [
    (1, 1, 100, 9700), (2, 20, 100, 10016), (1, 70, 37, 9700), (1, 5, 301, 12000),      # rows that LDS does not hold
    (1, 40, 100, 2048), (2, 33, 1000, 2000), (1, 16, 130, 9000)])                       # and those that take more than 64 KB of it
def test_project_of_few_tokens_and_wide_rows(dev, dtype, L, T, F, d):
    x = _whole_numbers((L, T, d), 0, T).to(dtype)
    w = _whole_numbers((L, F, d), 1, F)
    b = (torch.arange(L * F).reshape(L, F) % 200 - 100).to(dtype)
    want = (torch.bmm(x.double(), w.double().transpose(1, 2).contiguous()) + b.double().unsqueeze(1)).to(dtype)
    wq = cca.mx.quantise(w.to(dev))
    got = cca.mx.project(x.to(dev), wq, b.to(dev))
    assert torch.equal(got.cpu(), want)
    assert torch.equal(cca.mx.project(cca.mx.quantise(x.to(dev)), wq, b.to(dev)).cpu(), want)


def test_quantise_again_shows_a_write_that_the_samples_miss(dev):
    """Of a row 32 elements of 16 bits are looked at, of the first row the first ones."""
    model, inputs, x = _model(dev)
    model.quantise_encoder()
    with torch.no_grad():
        _true(model, inputs, x)
        model.encoder_module.encoders[1].weight.data[0, 100] = 50.0
        model.quantise_encoder()
        _true(model, inputs, x)
        model.encoder_module.encoders[2].weight[5, 77] = -50.0       # not past the version counter: shows by itself
        _true(model, inputs, x)
