"""Microscaled formats on the device: quantisation, the activation cache and the projection against the oracle in float64.

Tolerances.  Codes and scales are compared bit by bit, and so is what is read back without a normalisation where the type
holds it.  A normalised value takes one rounding of the difference, one of the quotient and one to the type: relative
2^-24 + 2^-24 + half a step.  A sum of K exact products in float32, in any order and with its additions rounded or cut
off, is within K 2^-23 of the sum of the products' magnitudes; the bias adds one more addition, the type half a step."""
import pytest
import torch

import crosslayer_coding_amd as cca
from oracle import mx_oracle as orc

pytestmark = pytest.mark.gpu

FORMATS = ["mxfp4", "mxfp8", "mxint8"]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rows(n, d, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g) * torch.exp(spread * torch.randn(n, 1, generator=g))
    x[:, torch.randint(0, d, (2,), generator=g)] *= 20.0
    ties = torch.randint(-16, 17, (n, d), generator=g).float() / 4          # values on and between grid points
    x = torch.where(torch.rand(n, 1, generator=g) < 0.3, ties, x)
    return x.clamp(-60000, 60000).to(dtype)


def _check_codes(q, x, fmt):
    codes, scales = orc.quantise(x, fmt)
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.codes.cpu(), codes)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 100), (64, 64), (130, 768), (33, 2048), (2, 4100)])
def test_quantise_and_back(dev, fmt, dtype, n, d):
    x = _rows(n, d, dtype, seed=n + d)
    q = cca.mx.quantise(x.to(dev), fmt)
    _check_codes(q, x, fmt)
    back = orc.round_trip(x, fmt)
    for out in DTYPES:
        assert torch.equal(q.dequantise(out).cpu(), back.float().to(out))


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_value_of_a_16_bit_type(dev, fmt):
    """All bf16 and fp16 bit patterns, each beside a value that fixes the scale, and alone in its block."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    for dtype in (torch.bfloat16, torch.float16):
        v = bits.view(dtype)
        alone = torch.zeros(65536, 32, dtype=dtype)
        alone[:, 7] = v
        beside = alone.clone()
        beside[:, 20] = 1.75
        for x in (alone, beside):
            _check_codes(cca.mx.quantise(x.to(dev), fmt), x, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_ends_of_float32(dev, fmt):
    tiny, top = 2.0 ** -149, torch.finfo(torch.float32).max
    vals = [0.0, -0.0, tiny, -tiny, 2.0 ** -127, 2.0 ** -126, 1.5 * 2.0 ** -126, 2.0 ** -120, top, -top, 2.0 ** 127, 1.0]
    x = torch.zeros(len(vals), 64)
    for i, v in enumerate(vals):
        x[i, 0], x[i, 33], x[i, 40] = v, v / 2, v * 0.3
    q = cca.mx.quantise(x.to(dev), fmt)
    _check_codes(q, x, fmt)
    assert torch.equal(q.dequantise().cpu().double(), orc.round_trip(x, fmt).float().double())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_block_without_a_number_reads_as_nan_and_no_other(dev, fmt, bad):
    x = _rows(6, 96, torch.float32)
    x[2, 40] = bad
    back = cca.mx.quantise(x.to(dev), fmt).dequantise().cpu()
    want = orc.round_trip(x, fmt).float()
    assert torch.isnan(back[2, 32:64]).all()
    assert torch.equal(back.isnan(), want.isnan()) and torch.equal(back.nan_to_num(), want.nan_to_num())


def test_strides_and_offsets(dev):
    base = _rows(40, 200, torch.bfloat16).to(dev)
    for x in (base[:, 8:136], base[::3, :64], base[:, 3:100], base[5:6], base.t()[:50], base[:, :1].expand(40, 40), base[1:, :192].reshape(3, 13, 192),
              base[:0]):
        q = cca.mx.quantise(x, "mxfp8")
        assert q.shape == x.shape
        if x.numel():
            _check_codes(q, x.contiguous(), "mxfp8")
    into = cca.mx.quantise(base, "mxfp4")
    again = cca.mx.quantise(base * 2, "mxfp4", out=into)
    assert again is into
    _check_codes(into, base * 2, "mxfp4")


# ---- the cache ---------------------------------------------------------------------------------------------------

def _cache(L, R, d, fmt, dev, seed=1):
    """A filled cache and the values it holds, float64 [L, 2, R, d]."""
    x = torch.stack([torch.stack([_rows(R, d, torch.float32, seed + 7 * l + k) for k in range(2)]) for l in range(L)])
    codes, scales = orc.quantise(x, fmt)
    return cca.MXActivationCache(codes.to(dev), scales.to(dev), fmt, d), orc.dequantise(codes, scales, fmt, d)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,R,d,n", [(1, 1, 1, 1), (2, 50, 64, 17), (3, 40, 100, 40), (12, 300, 768, 130), (2, 20, 33, 64)])
def test_read_gathers_and_normalises(dev, fmt, dtype, L, R, d, n):
    cache, held = _cache(L, R, d, fmt, dev)
    g = torch.Generator().manual_seed(5)
    rows = torch.randint(0, R, (n,), generator=g)
    tables = [t for _ in range(2) for t in (torch.randn(L, d, generator=g), torch.rand(L, d, generator=g) + 0.5)]
    for norm in ("none", "mean_std", "sqrt_d_model"):
        got = cache.read(rows.to(dev), dtype, norm, [t.to(dev) for t in tables] if norm == "mean_std" else None)
        for kind in range(2):
            want = held[:, kind][:, rows]
            steps = 0.0
            if norm == "mean_std":
                want = (want - tables[2 * kind].double().unsqueeze(1)) / tables[2 * kind + 1].double().unsqueeze(1)
                steps = 2 * 2.0 ** -24
            elif norm == "sqrt_d_model":
                want = want * d ** 0.5
                steps = 2 * 2.0 ** -24                      # the factor and the product
            info = torch.finfo(dtype)
            tol = want.abs() * (steps + info.eps / 2) * 1.01 + info.smallest_normal * info.eps / 2
            over = want.abs() > info.max
            assert got[kind].dtype == dtype and got[kind].shape == (L, n, d)
            err = (got[kind].cpu().double() - want).abs()
            assert bool(((err <= tol) | over).all()), (norm, kind, float((err / tol).max()))


def test_read_takes_rows_in_every_form(dev):
    cache, held = _cache(2, 30, 64, "mxint8", dev)
    want = held[:, :, 4:9].float()
    for rows in (slice(4, 9), range(4, 9), [4, 5, 6, 7, 8], torch.arange(4, 9), torch.arange(4, 9).numpy().astype("uint32"),
                 torch.arange(4, 9, device=dev), torch.arange(4, 9, device=dev, dtype=torch.int32), torch.arange(0, 18, device=dev)[8:18:2] // 2):
        x, tg = cache.read(rows, torch.float32)
        assert torch.equal(x.cpu(), want[:, 0]) and torch.equal(tg.cpu(), want[:, 1])
    assert cache.read([], torch.float32)[0].shape == (2, 0, 64)
    # into rows of a larger batch; the others stay
    out = (torch.full((2, 9, 64), 7.0, device=dev), torch.full((2, 9, 64), 7.0, device=dev))
    cache.read(slice(4, 9), torch.float32, out=out, out_row=3)
    for kind in range(2):
        assert torch.equal(out[kind][:, 3:8].cpu(), want[:, kind]) and bool((out[kind][:, :3] == 7).all()) and bool((out[kind][:, 8:] == 7).all())
    # one kind without statistics is left as it is
    t = torch.full((2, 64), 2.0, device=dev)
    x, tg = cache.read(slice(4, 9), torch.float32, "mean_std", (None, None, t, t))
    assert torch.equal(x.cpu(), want[:, 0]) and torch.equal(tg.cpu(), (want[:, 1] - 2) / 2)


def test_rows_outside_the_cache(dev):
    cache, held = _cache(2, 10, 64, "mxfp4", dev)
    rows = torch.tensor([3, -1, 10, 2 ** 40, 9], device=dev)
    x, tg = cache.read(rows, torch.float32)
    for got, want in ((x, held[:, 0]), (tg, held[:, 1])):
        assert torch.isnan(got[:, 1:4]).all()
        assert torch.equal(got[:, [0, 4]].cpu(), want[:, [3, 9]].float())
    before = cache.codes.clone(), cache.scales.clone()
    new = torch.ones(2, 5, 64, device=dev)
    cache.write(rows, new, new)
    keep = [r for r in range(10) if r not in (3, 9)]
    assert torch.equal(cache.codes[:, :, keep], before[0][:, :, keep]) and torch.equal(cache.scales[:, :, keep], before[1][:, :, keep])
    assert bool((cache.read([3, 9], torch.float32)[1] == 1).all())
    with pytest.raises(IndexError):
        cache.write([3, 10], new[:, :2], new[:, :2])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["run", "device", "host"])
@pytest.mark.parametrize("L,R,d,n", [(1, 5, 32, 1), (3, 60, 100, 19), (2, 300, 768, 257)])
def test_write_changes_its_rows_and_no_others(dev, fmt, dtype, how, L, R, d, n):
    cache, _ = _cache(L, R, d, fmt, dev)
    codes, scales = cache.codes.cpu().clone(), cache.scales.cpu().clone()
    x, tg = (torch.stack([_rows(n, d, dtype, 50 + 2 * l + k) for l in range(L)]) for k in range(2))
    g = torch.Generator().manual_seed(3)
    rows = torch.arange(2, 2 + n) if how == "run" else torch.randperm(R, generator=g)[:n]
    cache.write(slice(2, 2 + n) if how == "run" else rows.to(dev) if how == "device" else rows.numpy(), x.to(dev), tg.to(dev))
    for kind, v in ((0, x), (1, tg)):
        c, s = orc.quantise(v, fmt)
        codes[:, kind, rows], scales[:, kind, rows] = c, s
    assert torch.equal(cache.codes.cpu(), codes) and torch.equal(cache.scales.cpu(), scales)


def test_a_row_named_twice_keeps_the_later_one(dev):
    L, R, d, n = 2, 64, 96, 1000
    cache = cca.MXActivationCache.empty(L, R, d, "mxfp8", dev)
    assert torch.isnan(cache.read(slice(None))[0]).all()            # nothing has been written
    g = torch.Generator().manual_seed(2)
    for trial in range(3):
        rows = torch.randint(0, R, (n,), generator=g)
        x = torch.stack([_rows(n, d, torch.bfloat16, trial + l) for l in range(L)])
        cache.write(rows.to(dev), x.to(dev), (2 * x).to(dev))
        last = {int(r): j for j, r in enumerate(rows)}
        at, src = list(last), [last[r] for r in last]
        got = cache.read(at, torch.bfloat16)
        assert torch.equal(got[0].cpu(), orc.round_trip(x[:, src], "mxfp8").to(torch.bfloat16))
        assert torch.equal(got[1].cpu(), orc.round_trip(2 * x[:, src], "mxfp8").to(torch.bfloat16))


def test_write_takes_layers_apart_and_strided_batches(dev):
    L, d = 3, 64
    cache = cca.MXActivationCache.empty(L, 40, d, "mxint8", dev)
    x = torch.stack([_rows(20, d, torch.bfloat16, l) for l in range(L)]).to(dev)
    want = orc.round_trip(x, "mxint8").to(torch.bfloat16)
    cache.write(slice(0, 20), {l: x[l].clone() for l in range(L)}, {l: x[l].reshape(4, 5, d) for l in range(L)})
    got = cache.read(slice(0, 20))
    assert torch.equal(got[0].cpu(), want) and torch.equal(got[1].cpu(), want)
    big = torch.zeros(L, 40, 2 * d, dtype=torch.bfloat16, device=dev)
    big[:, ::2, :d] = x
    cache.write(range(20, 40), big[:, ::2, :d], x)
    got = cache.read(slice(20, 40))
    assert torch.equal(got[0].cpu(), want) and torch.equal(got[1].cpu(), want)
    cache.write([7], x[:, :1].expand(L, 1, d), x[:, :1])
    cache.write(slice(0, 0), x[:, :0], x[:, :0])
    assert torch.equal(cache.read([7])[0].cpu(), want[:, :1])
    with pytest.raises(ValueError):
        cache.write(slice(0, 3), x[:, :3], x[:, :4])
    with pytest.raises(ValueError):
        cache.write(slice(0, 3), x[:, :3], x[:, :3].float())
    with pytest.raises(ValueError):
        cache.write(slice(0, 3), {0: x[0, :3]}, x[:, :3])


def test_offsets_beyond_32_bits(dev):
    """5 GB of codes: the last rows of the last layer lie past what 32 bits address."""
    L, R, d = 2, 1700000, 768
    cache = cca.MXActivationCache.empty(L, R, d, "mxfp8", dev)
    assert cache.codes.numel() > 2 ** 32
    x = torch.stack([_rows(9, d, torch.bfloat16, l) for l in range(L)])
    want = orc.round_trip(x, "mxfp8").to(torch.bfloat16)
    cache.write(slice(R - 9, R), x.to(dev), (-x).to(dev))
    got = cache.read(torch.arange(R - 9, R, device=dev))
    assert torch.equal(got[0].cpu(), want) and torch.equal(got[1].cpu(), -want)
    assert torch.isnan(cache.read(slice(R - 10, R - 9))[1]).all() and torch.isnan(cache.read(slice(0, 2))[0]).all()


# ---- the projection ----------------------------------------------------------------------------------------------

def _check_project(got, xq, wq, b, dtype, rows=None):
    """xq, wq: the values the codes stand for."""
    K = wq.shape[-1]
    want = xq @ wq.transpose(-1, -2)
    mag = xq.abs() @ wq.abs().transpose(-1, -2)
    if b is not None:
        want = want + b.double().unsqueeze(-2)
        mag = mag + b.double().abs().unsqueeze(-2)
    tol = mag * (K + 1) * 2.0 ** -23 + want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def _weights(L, F, d, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = cca.mx.quantise(((torch.rand(L, F, d, generator=g) * 2 - 1) / d ** 0.5).to(dev), "mxfp4")
    return w, orc.dequantise(w.codes, w.scales, "mxfp4", d)


def _inputs(L, T, d, dtype, seed=0):
    return torch.stack([_rows(T, d, dtype, seed + l, spread=0.5) for l in range(L)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,T,d,F", [
    (1, 1, 1, 1), (1, 1, 32, 16), (2, 1, 768, 1000), (3, 5, 100, 37), (1, 16, 128, 64), (2, 17, 160, 250), (1, 33, 33, 260),
    (2, 77, 768, 1024), (1, 128, 640, 301), (1, 129, 256, 256), (2, 255, 512, 260), (1, 256, 768, 256), (2, 257, 640, 516),
    (1, 300, 1024, 1000), (1, 513, 2048, 772), (1, 256, 96, 255), (3, 260, 256, 2048), (1, 700, 1280, 1026)])
def test_project(dev, dtype, L, T, d, F):
    x = _inputs(L, T, d, dtype, T + F)
    w, wq = _weights(L, F, d, dev, d)
    g = torch.Generator().manual_seed(9)
    b = torch.randn(L, F, generator=g).to(dtype)
    xq = orc.round_trip(x, "mxfp4")
    got = cca.mx.project(x.to(dev), w, b.to(dev))
    assert got.dtype == dtype and got.shape == (L, T, F)
    _check_project(got, xq, wq, b, dtype)
    _check_project(cca.mx.project(x.to(dev), w), xq, wq, None, dtype)


def test_project_adds_exactly_what_is_exact(dev):
    """Small whole numbers: every partial sum is exact, so any order gives the same result - each row, feature and
    element of K is told from its neighbours."""
    for T, d, F in ((1, 256, 300), (40, 320, 260), (300, 768, 520), (260, 2048, 1024), (513, 640, 772)):
        g = torch.Generator().manual_seed(T)
        x = torch.randint(-3, 4, (1, T, d), generator=g).float()
        x[..., ::32] = 6.0                                          # every block's scale is 1
        w = torch.randint(-3, 4, (1, F, d), generator=g).float()
        w[..., 1::32] = 4.0
        scale = torch.tensor([1.0, 2.0, 0.5, 8.0])[torch.randint(0, 4, (1, F, d // 32), generator=g)]
        w = (w.unflatten(-1, (-1, 32)) * scale.unsqueeze(-1)).flatten(-2)
        got = cca.mx.project(x.to(dev), cca.mx.quantise(w.to(dev)), torch.arange(F).float().unsqueeze(0).to(dev))
        want = x.double() @ w.double().transpose(1, 2) + torch.arange(F).double()
        assert torch.equal(got.cpu().double(), want), (T, d, F)


@pytest.mark.parametrize("T", [1, 40, 300])
def test_project_range_of_scales(dev, T):
    """Blocks from the smallest to the largest scale, within what float32 sums hold."""
    d, F = 256, 260
    x = _inputs(1, T, d, torch.float32)
    x = (x.unflatten(-1, (-1, 32)) * (2.0 ** torch.tensor([-100.0, -60, -20, 0, 20, 40, 60, 80])).unsqueeze(-1)).flatten(-2)
    g = torch.Generator().manual_seed(1)
    w = torch.rand(1, F, d, generator=g) * 2 - 1
    w = (w.unflatten(-1, (-1, 32)) * (2.0 ** -torch.tensor([-20.0, -60, -20, 0, 20, 40, 60, 90])).unsqueeze(-1)).flatten(-2)
    wq = cca.mx.quantise(w.to(dev))
    _check_project(cca.mx.project(x.to(dev), wq), orc.round_trip(x, "mxfp4"), orc.dequantise(wq.codes, wq.scales, "mxfp4", d), None, torch.float32)


@pytest.mark.parametrize("T,F,d", [(3, 100, 96), (300, 520, 640), (300, 520, 96), (300, 512, 768)])
def test_project_of_a_bad_token_or_feature_is_nan_and_no_other(dev, T, F, d):
    x = _inputs(1, T, d, torch.float32)
    x[0, 1, d - 1] = float("inf")
    w, _ = _weights(1, F, d, dev)
    w.scales[0, 5, 0] = 255
    got = cca.mx.project(x.to(dev), w).cpu()[0]
    bad = torch.zeros(T, F, dtype=torch.bool)
    bad[1], bad[:, 5] = True, True
    assert torch.equal(got.isnan(), bad)
    y = x.clone()
    y[0, 1, d - 1] = 0.0
    w.scales[0, 5, 0] = 100
    clean = cca.mx.project(y.to(dev), w).cpu()[0]
    assert torch.equal(got[~bad], clean[~bad])


def test_project_forms(dev):
    x = _inputs(2, 40, 192, torch.bfloat16)
    w, wq = _weights(2, 100, 192, dev)
    want = cca.mx.project(x.to(dev), w)
    one = cca.mx.project(x[1].to(dev), cca.MXTensor(w.codes[1].contiguous(), w.scales[1].contiguous(), "mxfp4", 192))
    assert torch.equal(one, want[1])
    xq = cca.mx.quantise(x.to(dev))
    assert torch.equal(cca.mx.project(xq, w, dtype=torch.bfloat16), want)
    out = torch.empty_like(want)
    assert cca.mx.project(xq, w, out=out) is out and torch.equal(out, want)
    b = torch.randn(100, 2, device=dev).to(torch.bfloat16).t()              # a bias that is not contiguous
    _check_project(cca.mx.project(xq, w, b), orc.round_trip(x, "mxfp4"), wq, b.cpu(), torch.bfloat16)
    assert cca.mx.project(x[:, :0].to(dev), w).shape == (2, 0, 100)
    _check_project(cca.mx.project(x.to(dev), w.index_select(torch.tensor([1, 0], device=dev))), orc.round_trip(x, "mxfp4"), wq[[1, 0]], None, torch.bfloat16)
    for bad in (b.float(), b[:1]):
        with pytest.raises(ValueError):
            cca.mx.project(x.to(dev), w, bad)
    with pytest.raises(ValueError):
        cca.mx.project(x.to(dev), w, out=out[:, :, :50])
    with pytest.raises(ValueError):
        cca.mx.project(x.to(dev), w, dtype=torch.float32)
    with pytest.raises(NotImplementedError):
        cca.mx.project(x.to(dev).requires_grad_(), w)
    with torch.no_grad():
        assert torch.equal(cca.mx.project(x.to(dev).requires_grad_(), w), want)


def test_project_is_the_same_every_time(dev):
    """One order of summation: calls repeat bit by bit."""
    for T in (1, 77, 1030):
        x = _inputs(2, T, 768, torch.bfloat16).to(dev)
        w, _ = _weights(2, 1000, 768, dev)
        first = cca.mx.project(x, w)
        for _ in range(5):
            assert torch.equal(cca.mx.project(x, w), first)


def test_project_of_more_outputs_than_32_bits_count(dev):
    L, T, F, d = 2, 16500, 66000, 32
    x = _inputs(1, T, d, torch.bfloat16)
    xl = x.expand(L, T, d).contiguous()
    w, wq = _weights(1, F, d, dev)
    w2 = w.index_select(torch.tensor([0, 0], device=dev))
    got = cca.mx.project(xl.to(dev), w2)
    assert got.numel() > 2 ** 31
    xq = orc.round_trip(x, "mxfp4")
    at = torch.tensor([0, 1, T // 2, T - 2, T - 1])
    _check_project(got[1][at.to(dev)], xq[0][at], wq[0], None, torch.bfloat16)
    _check_project(got[1][:, -300:], xq[0], wq[0][-300:], None, torch.bfloat16)
    assert torch.equal(got[0], got[1])


# ---- together ----------------------------------------------------------------------------------------------------

def _together(cache, rows, x, w, b):
    cache.write(rows, x, x)
    a, _ = cache.read(rows, torch.bfloat16, "sqrt_d_model")
    return cca.mx.project(a, w, b)


def test_on_another_stream(dev):
    L, T, d, F = 2, 100, 256, 300
    w, _ = _weights(L, F, d, dev)
    b = torch.randn(L, F, device=dev).to(torch.bfloat16)
    x = _inputs(L, T, d, torch.bfloat16).to(dev)
    rows = torch.randperm(500, device=dev)[:T]
    cache = cca.MXActivationCache.empty(L, 500, d, "mxfp8", dev)
    want = _together(cache, rows, x, w, b)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [_together(cache, rows, x, w, b) for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("T", [1, 70, 300])
def test_captured_and_replayed(dev, T):
    """A harvest step, a batch and its pre-activations in one graph, replayed on new contents between eager calls."""
    L, d, F, R = 2, 768, 516, 400
    w, _ = _weights(L, F, d, dev)
    b = torch.randn(L, F, device=dev).to(torch.bfloat16)
    x = _inputs(L, T, d, torch.bfloat16).to(dev)
    rows = torch.randperm(R, device=dev)[:T]
    cache = cca.MXActivationCache.empty(L, R, d, "mxfp4", dev)
    other = cca.MXActivationCache.empty(L, R, d, "mxfp4", dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _together(cache, rows, x, w, b)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = _together(cache, rows, x, w, b)
    for trial in range(4):
        x.copy_(_inputs(L, T, d, torch.bfloat16, 11 * trial).to(dev))
        rows.copy_(torch.randperm(R, device=dev)[:T])
        g.replay()
        want = _together(other, rows, x, w, b)
        torch.cuda.synchronize()
        assert torch.equal(got, want), trial


# ---- weights that were written -----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,n,d", [(1, 1, 1), (2, 7, 33), (3, 300, 100), (2, 4100, 256), (2, 130, 2050)])
def test_refresh_follows_writes_to_any_row_column_or_layer(dev, dtype, L, n, d):
    g = torch.Generator().manual_seed(n)
    w = torch.randn(L, n, d, generator=g).to(dtype).to(dev)
    q = cca.mx.quantise(w)
    state, changed = torch.zeros(16 * L, dtype=torch.int64, device=dev), torch.zeros(L, dtype=torch.int32, device=dev)
    cca.mx.refresh(w, q, state, changed, store_only=True)
    cca.mx.refresh(w, q, state, changed)
    assert changed.tolist() == [0] * L
    for trial in range(4):
        l, r, c = int(torch.randint(L, (1,), generator=g)), int(torch.randint(n, (1,), generator=g)), int(torch.randint(d, (1,), generator=g))
        for write in (lambda: w[l, r].mul_(-1.5), lambda: w[l, :, c].add_(0.75), lambda: w[l].mul_(0.5)):
            write()
            cca.mx.refresh(w, q, state, changed)
            assert changed.tolist() == [int(i == l) for i in range(L)]
            _check_codes(q, w.cpu(), "mxfp4")
            cca.mx.refresh(w, q, state, changed)
            assert not changed.any()


def test_an_output_inside_the_input_is_refused(dev):
    w = cca.mx.quantise(torch.randn(256, 256, device=dev))
    buf = torch.randn(80, 256, device=dev)
    before = buf.clone()
    for a, b in ((0, 0), (0, 20), (20, 0)):
        with pytest.raises(ValueError, match="out lies in x"):
            cca.mx.project(buf[a:a + 40], w, out=buf[b:b + 40])
    assert torch.equal(buf, before)
    assert torch.equal(cca.mx.project(buf[:40], w, out=buf[40:]), cca.mx.project(before[:40], w))
    strided = torch.randn(40, 512, device=dev)[:, ::2]
    assert torch.equal(cca.mx.project(strided, w), cca.mx.project(strided.contiguous(), w))


@pytest.mark.parametrize("first,n", [(0, 3), (1, 1), (2, 1), (1, 2)])
def test_narrowed_weights_are_the_layers_themselves(dev, first, n):
    q = cca.mx.quantise(torch.randn(3, 300, 100, device=dev))
    x = torch.randn(n, 5, 100, device=dev)
    part = q.narrow(first, n)
    assert part.codes.data_ptr() == q.codes[first].data_ptr() and part.shape == (n, 300, 100)
    assert torch.equal(cca.mx.project(x, part), cca.mx.project(x, q.index_select(torch.arange(first, first + n, device=dev))))
