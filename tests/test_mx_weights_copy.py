"""The 4-bit copy of a quantised encoder's weights: when it is made, looked at and kept, on the host.

The device is played by lists of launches.  An eager launch runs at once; one under a capture is put down with what a graph
would have of it - addresses, which keep nothing alive - and runs when it is replayed."""
import weakref

import numpy as np
import pytest
import torch

import crosslayer_coding_amd as cca
from crosslayer_coding_amd import encoder as encoder_module
from oracle import mx_oracle as orc

L, D, F = 3, 64, 40


class Device:
    def __init__(self):
        self.recording = None
        self.quantised = 0

    def launch(self, run, *memory):
        """``run(*memory)``; memory: tensors that the launch has the addresses of."""
        if self.recording is None:
            run(*memory)
            return
        refs = [weakref.ref(t) for t in memory]

        def replay():
            held = [r() for r in refs]
            assert all(t is not None for t in held), "a captured launch goes to memory that was given back"
            run(*held)

        self.recording.append(replay)

    def capture(self, call):
        self.recording, graph = [], None
        call()
        graph, self.recording = self.recording, None
        return graph

    # ---- mx.quantise and mx.refresh, from the oracle; every element counts in these fingerprints
    def quantise(self, x, fmt, out=None):
        if out is None:
            pitch, blocks = cca.mx.row_layout(x.shape[-1], fmt)
            out = cca.MXTensor(torch.zeros(*x.shape[:-1], pitch, dtype=torch.uint8), torch.zeros(*x.shape[:-1], blocks, dtype=torch.uint8), fmt, x.shape[-1])

        def run(codes, scales):
            self.quantised += 1
            c, s = orc.quantise(x, fmt)
            codes.copy_(c), scales.copy_(s)

        self.launch(run, out.codes, out.scales)
        return out

    def refresh(self, x, out, state, changed, store_only=False, first=0, n=None):
        def run(codes, scales, state, changed):
            for l in range(first, L if n is None else first + n):
                line = state[16 * l:16 * l + 3]
                assert int(line[0]) == 0 and int(line[1]) == 0, "sum and arrivals begin at zero"
                now = int(np.frombuffer(x[l].contiguous().numpy().tobytes(), dtype=np.uint32).astype(np.int64).cumsum().sum() % (2 ** 62))
                changed[l] = int(not store_only and int(line[2]) != now)
                line[2] = now
                if changed[l]:
                    c, s = orc.quantise(x[l], "mxfp4")
                    codes[l].copy_(c), scales[l].copy_(s)

        self.launch(run, out.codes, out.scales, state, changed)


@pytest.fixture
def device(monkeypatch):
    d = Device()
    monkeypatch.setattr(encoder_module.mx, "quantise", d.quantise)
    monkeypatch.setattr(encoder_module.mx, "refresh", d.refresh)
    monkeypatch.setattr(encoder_module.nat, "require_device", lambda t, what: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: d.recording is not None)
    return d


@pytest.fixture
def enc(device):
    cfg = cca.CLTConfig(num_features=F, num_layers=L, d_model=D, batchtopk_k=4, clt_dtype="float32")
    e = encoder_module.Encoder(cfg, None, torch.device("cpu"), torch.float32)
    g = torch.Generator().manual_seed(3)
    with torch.no_grad():
        for lin in e.encoders:
            lin.weight.copy_(torch.randn(F, D, generator=g))
    e.quantise()
    return e


def _true(enc, layers=range(L)):
    q = enc._mx
    for l in layers:
        codes, scales = orc.quantise(enc.encoders[l].weight.detach(), "mxfp4")
        assert torch.equal(q.codes[l], codes) and torch.equal(q.scales[l], scales), l


def _write(enc, l, how):
    w = enc.encoders[l].weight
    with torch.no_grad():
        if how == "mul_":
            w.mul_(-1.5)
        elif how == "load_state_dict":
            enc.load_state_dict({k: v * 0.5 for k, v in enc.state_dict().items()})
        else:
            w.data.mul_(2.0)


@pytest.mark.parametrize("how", ["mul_", "load_state_dict"])
@pytest.mark.parametrize("between", ["eager", "capture"])
def test_fingerprints_outlive_the_writes_that_a_captured_forward_lives_through(device, enc, how, between):
    enc.quantised_weights()
    graph = device.capture(enc.quantised_weights)
    for trial in range(2):
        _write(enc, 1, how)
        if between == "eager":
            enc.quantised_weights()
        else:
            device.capture(enc.quantised_weights)
            enc.quantised_weights()
        _write(enc, 2, "data")
        for launch in graph:
            launch()
        _true(enc)
        enc.quantised_weights()
        _true(enc)


@pytest.mark.parametrize("layers", ["all", "one"])
def test_a_write_while_nobody_watched_is_seen_when_somebody_does_again(device, enc, layers):
    enc.watch_parameter_data = False
    _write(enc, 1, "mul_")
    enc.quantised_weights()                             # made without a look at the data
    _true(enc)
    for l in range(L):
        _write(enc, l, "data")
    enc.quantised_weights()
    enc.watch_parameter_data = True
    if layers == "one":
        enc._quantised_slab(2, 1)
        _true(enc, [2])
    enc.quantised_weights()
    _true(enc)


def test_watching_from_the_first_copy_on_is_not_needed(device, enc):
    enc.dequantise()
    enc.watch_parameter_data = False
    enc.quantise()
    _write(enc, 0, "data")
    enc.watch_parameter_data = True
    enc.quantised_weights()
    _true(enc)
    before = device.quantised
    enc.quantised_weights()
    assert device.quantised == before


def test_a_replay_that_makes_the_copy_takes_its_fingerprints_too(device, enc):
    """Weights put in for one replay and taken out again, all past the version counters."""
    _write(enc, 1, "mul_")
    graph = device.capture(enc.quantised_weights)       # right after a write: the graph quantises
    enc.quantised_weights()
    kept = enc.encoders[1].weight.detach().clone()
    enc.encoders[1].weight.data.mul_(0.3)
    for launch in graph:
        launch()
    _true(enc)
    enc.encoders[1].weight.data.copy_(kept)
    enc.quantised_weights()
    _true(enc)


def test_a_copy_that_is_first_made_under_a_capture(device, enc):
    enc.dequantise()
    enc._mx_fmt = "mxfp4"                               # as after a move to another device: there is no copy there yet
    graphs = [device.capture(enc.quantised_weights) for _ in range(2)]
    for trial in range(2):
        _write(enc, 1, "data")
        for launch in graphs[trial]:
            launch()
        _true(enc)
    _write(enc, 2, "data")
    enc.quantised_weights()
    _true(enc)
    _write(enc, 0, "data")
    enc.quantised_weights()
    _true(enc)


def test_a_copy_that_cannot_be_made_leaves_the_encoder_as_it_was(device, enc, monkeypatch):
    def no_memory(*args, **kw):
        raise torch.cuda.OutOfMemoryError("no memory for the copy")

    enc.dequantise()
    with monkeypatch.context() as m:
        m.setattr(encoder_module.mx, "quantise", no_memory)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            enc.quantise()
        assert enc.quantised is None and enc._mx is None
    enc.quantise()
    _true(enc)
    with pytest.raises(ValueError):
        enc.quantise("mxfp8")
    _write(enc, 0, "mul_")
    with monkeypatch.context() as m:                    # a copy that is there stays in use, and is made anew when it can be
        m.setattr(encoder_module.mx, "quantise", no_memory)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            enc.quantise()
    assert enc.quantised == "mxfp4"
    enc.quantised_weights()
    _true(enc)


@pytest.mark.parametrize("layers", [[1], [0, 1], [0, 2]])
def test_some_layers_of_a_quantised_encoder_copy_no_weights_that_nobody_reads(device, enc, monkeypatch, layers):
    inputs = {l: torch.randn(5, D) for l in layers}
    slab = enc._w_slab.untyped_storage().data_ptr()
    enc.dequantise()
    assert enc.prepare_slab(inputs)[2].shape == (len(layers), F, D)
    enc.quantise()
    got, x, w, b = enc.prepare_slab(inputs)
    assert got == layers and x.shape == (len(layers), 5, D)
    assert w.untyped_storage().data_ptr() == slab
    assert torch.equal(b, enc._b_slab[layers])
    seen = []
    monkeypatch.setattr(encoder_module.mx, "project", lambda x, q, b, out=None, ws=None: seen.append(q) or torch.zeros(*x.shape[:2], F))
    _, pre = enc.encode_slab(inputs)
    codes, scales = orc.quantise(enc._w_slab[layers].detach(), "mxfp4")
    assert pre.shape == (len(layers), 5, F) and torch.equal(seen[0].codes, codes) and torch.equal(seen[0].scales, scales)


def test_quantise_again_makes_the_copy_anew_where_it_is(device, enc):
    """For writes that a look at samples of the data may miss; captured forwards go on with the copy."""
    graph = device.capture(enc.quantised_weights)
    at, before = enc._mx.codes.data_ptr(), device.quantised
    enc.quantise()
    assert device.quantised == before + 1 and enc._mx.codes.data_ptr() == at
    _write(enc, 0, "data")
    for launch in graph:
        launch()
    _true(enc)
