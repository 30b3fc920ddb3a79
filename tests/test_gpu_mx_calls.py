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
    pre, _ = model._encode_all_layers(inputs)
    # half a step of the type that the results have: a model that was just moved to another type knows its own with the next call
    tol = (xq.abs() @ wq.abs().transpose(1, 2) + b.abs()) * (w.shape[-1] + 1) * 2.0 ** -23 + want.abs() * torch.finfo(pre[0].dtype).eps / 2 * 1.01 + 1e-30
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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,T,F,d,row,gap,at", [
    (2, 300, 520, 320, 528, 64, 0), (2, 300, 512, 640, 576, 0, 64), (1, 77, 257, 768, 260, 0, 2), (2, 5, 100, 96, 101, 7, 1),
    (2, 513, 301, 160, 301, 3, 1), (3, 600, 768, 256, 1024, 256, 0), (1, 64, 1000, 2048, 1001, 0, 0)])
def test_project_into_rows_of_a_larger_buffer(dev, dtype, L, T, F, d, row, gap, at):
    """The C entry: rows ``row`` elements apart, layers ``gap`` more, the first at an address of its own; what lies between stays."""
    lib = cca._native.load()
    x = _whole_numbers((L, T, d), 0, T).to(dtype).to(dev)
    w = cca.mx.quantise(_whole_numbers((L, F, d), 1, F).to(dev))
    b = (torch.arange(L * F).reshape(L, F) % 200 - 100).to(dtype).to(dev)
    layer = T * row + gap
    buf = torch.full((at + L * layer + 500,), 7.0, dtype=dtype, device=dev)
    nbytes = lib.clt_mx_encode_workspace_bytes(T, d, F, L, 0)
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
    code = lib.clt_mx_encode(x.data_ptr(), None, w.codes.data_ptr(), w.scales.data_ptr(), b.data_ptr(), buf.data_ptr() + at * buf.element_size(),
                             T, d, F, L, T * d, F, layer, row, cca._native.dtype_code(dtype), ws.data_ptr(), nbytes, cca._native.current_stream(dev))
    assert code == 0
    want = torch.full_like(buf, 7.0)
    w64 = w.dequantise().double()
    for l in range(L):
        pre = (torch.mm(x[l].double(), w64[l].t().contiguous()) + b[l].double()).to(dtype)
        want[at + l * layer:at + l * layer + T * row].view(T, row)[:, :F] = pre
    assert torch.equal(buf, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8", "mxint8"])
@pytest.mark.parametrize("n,d,row,at", [(9, 96, 96, 1), (300, 64, 72, 0), (5, 100, 103, 3), (2000, 768, 1024, 0), (1500, 768, 776, 8), (1, 33, 0, 5)])
def test_rows_apart_and_at_any_address_come_and_go(dev, dtype, fmt, n, d, row, at):
    """The C entries: quantised from rows of a larger buffer, given out into rows of another, which keeps what lies between."""
    lib = cca._native.load()
    code, stream = cca._native.dtype_code(dtype), cca._native.current_stream(dev)
    g = torch.Generator().manual_seed(n + d)
    src = torch.randn(at + n * max(row, d) + 64, generator=g).to(dtype).to(dev)
    pitch, blocks = cca.mx.row_layout(d, fmt)
    codes = torch.full((n + 1, pitch), 9, dtype=torch.uint8, device=dev)
    scales = torch.full((n + 1, blocks), 9, dtype=torch.uint8, device=dev)
    f = cca.mx.FORMATS[fmt]
    assert lib.clt_mx_quantise(src.data_ptr() + at * src.element_size(), n, d, row, code, f, codes.data_ptr(), scales.data_ptr(), stream) == 0
    rows = src[at:].as_strided((n, d), (max(row, d) if n > 1 else d, 1), at).cpu()
    c, s = orc.quantise(rows, fmt)
    assert torch.equal(codes[:n].cpu(), c) and torch.equal(scales[:n].cpu(), s)
    assert bool((codes[n] == 9).all()) and bool((scales[n] == 9).all())
    out = torch.full_like(src, 7.0)
    assert lib.clt_mx_dequantise(codes.data_ptr(), scales.data_ptr(), n, d, f, out.data_ptr() + at * out.element_size(), row, code, stream) == 0
    want = torch.full_like(src, 7.0)
    want.as_strided((n, d), (max(row, d) if n > 1 else d, 1), at).copy_(orc.dequantise(c, s, fmt, d).to(dtype))
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("fn", ["batchtopk", "topk", "jumprelu", "relu"])
def test_captured_forwards_of_every_activation(dev, fn, dtype):
    model, inputs, x = _model(dev, T=70, dtype=dtype, fn=fn)
    model.quantise_encoder()
    with torch.no_grad():
        g, out = _capture(model, inputs)
        for trial in range(3):
            x.copy_(torch.roll(x, 1, dims=1) * 1.25)
            if trial == 1:
                model.encoder_module.encoders[2].weight.data.mul_(0.5)
            if trial == 2:
                model.encoder_module.encoders[0].weight.mul_(-1.0)
            g.replay()
            torch.cuda.synchronize()
            got = {l: v.clone() for l, v in out.items()}
            pre, _ = model._encode_all_layers(inputs)
            want = model(inputs)
            for l in got:
                # eager threshold models may decode by another route, which adds in another order
                scale = float(want[l].float().abs().max())
                assert float((got[l].float() - want[l].float()).abs().max()) <= (2.0 ** -6 if fn in ("jumprelu", "relu") else 0.0) * scale, (trial, l)
        _true(model, inputs, x)


def test_a_copied_model_has_a_copy_of_its_own(dev):
    import copy

    model, inputs, x = _model(dev)
    model.quantise_encoder()
    with torch.no_grad():
        want = {l: v.clone() for l, v in model(inputs).items()}
        twin = copy.deepcopy(model)
        twin.encoder_module.encoders[1].weight.data.neg_()
        _true(twin, inputs, x)
        _true(model, inputs, x)
        twin.dequantise_encoder()
        again = model(inputs)
        assert all(torch.equal(again[l], want[l]) for l in want)


def test_a_model_of_another_type_or_device_and_back(dev):
    model, inputs, x = _model(dev, dtype="float32")
    model.quantise_encoder()
    with torch.no_grad():
        model(inputs)
        model.to(torch.bfloat16)
        _true(model, {l: v.bfloat16() for l, v in inputs.items()}, x.bfloat16())
        model.cpu()
        model.encoder_module.encoders[0].weight.data.neg_()
        model.to(dev)
        _true(model, {l: v.bfloat16() for l, v in inputs.items()}, x.bfloat16())
