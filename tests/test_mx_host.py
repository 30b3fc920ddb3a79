"""Microscaled formats on the host: layout, refusals, and the oracle against torch's own e4m3 type."""
import os
import re
import shutil
import subprocess

import pytest
import torch

import crosslayer_coding_amd as cca
from crosslayer_coding_amd import _native as nat
from crosslayer_coding_amd import build as clt_build
from oracle import mx_oracle as orc


def _held(lead, d, fmt="mxfp4"):
    pitch, blocks = cca.mx.row_layout(d, fmt)
    return torch.zeros(*lead, pitch, dtype=torch.uint8), torch.zeros(*lead, blocks, dtype=torch.uint8)


def test_row_layout_agrees_with_the_library():
    lib = nat.load()
    for fmt, code in cca.mx.FORMATS.items():
        for d in (1, 31, 32, 33, 100, 768, 2048, 262144):
            pitch, blocks = cca.mx.row_layout(d, fmt)
            assert lib.clt_mx_row_bytes(d, code) == pitch and blocks == (d + 31) // 32
    assert lib.clt_mx_row_bytes(0, 0) == 0 and lib.clt_mx_row_bytes(32, 3) == 0
    with pytest.raises(ValueError):
        cca.mx.row_layout(262145, "mxfp8")
    with pytest.raises(ValueError):
        cca.mx.row_layout(32, "fp4")


def test_oracle_rounds_like_the_e4m3_type():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 96, generator=g) * torch.exp(2 * torch.randn(64, 1, generator=g))
    codes, scales = orc.quantise(x, "mxfp8")
    up = torch.ldexp(x.double().unflatten(-1, (-1, 32)), (127 - scales.to(torch.int64)).unsqueeze(-1)).flatten(-2)
    want = up.float().clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(codes, want.view(torch.uint8))


def test_oracle_known_answers():
    x = torch.zeros(1, 32)
    x[0, :8] = torch.tensor([6.0, 5.0, -2.5, 0.25, 0.75, -0.2, 3.5, -7.9])
    codes, scales = orc.quantise(x, "mxfp4")            # largest 7.9: exponent 2, scale 1
    assert int(scales[0, 0]) == 127
    assert orc.dequantise(codes, scales, "mxfp4", 32)[0, :8].tolist() == [6.0, 4.0, -2.0, 0.0, 1.0, -0.0, 4.0, -6.0]
    codes, scales = orc.quantise(x, "mxint8")           # scale 2^2, steps of 4 / 64
    assert int(scales[0, 0]) == 129
    assert orc.dequantise(codes, scales, "mxint8", 32)[0, :3].tolist() == [6.0, 5.0, -2.5]
    assert float(orc.dequantise(codes, scales, "mxint8", 32)[0, 7]) == -7.875       # 126.4 steps of 1/16
    assert orc.quantise(torch.zeros(1, 5), "mxfp8")[1].tolist() == [[0]]
    assert orc.quantise(torch.tensor([[1.0, float("inf")]]), "mxfp8")[1].tolist() == [[255]]


def test_tensor_refusals():
    codes, scales = _held((4,), 100)
    cca.MXTensor(codes, scales, "mxfp4", 100)
    for bad in ((codes, scales, "mxfp4", 128 + 32), (codes, scales, "mxfp8", 100), (codes[:3], scales, "mxfp4", 100),
                (codes.to(torch.int8), scales, "mxfp4", 100), (codes[:, :32], scales, "mxfp4", 64), (codes, scales, "nf4", 100),
                (codes, scales, "mxfp4", 0)):
        with pytest.raises(ValueError):
            cca.MXTensor(*bad)
    flat = torch.zeros(4 * 64 + 16, dtype=torch.uint8)
    at = next(o for o in range(1, 16) if (flat.data_ptr() + o) % 16 != 0)
    with pytest.raises(ValueError, match="16 bytes"):
        cca.MXTensor(flat[at:at + 256].view(4, 64), scales, "mxfp4", 100)


def test_there_is_no_cpu_path():
    codes, scales = _held((2, 4), 64)
    w = cca.MXTensor(codes, scales, "mxfp4", 64)
    with pytest.raises(nat.CLTNativeError):
        cca.mx.quantise(torch.zeros(3, 64))
    with pytest.raises(nat.CLTNativeError):
        w.dequantise()
    with pytest.raises(nat.CLTNativeError):
        cca.mx.project(torch.zeros(2, 3, 64), w)
    cache = cca.MXActivationCache.empty(2, 8, 64, "mxfp8", device="cpu")
    with pytest.raises(nat.CLTNativeError):
        cache.read([0, 1])
    with pytest.raises(nat.CLTNativeError):
        cache.write([0, 1], torch.zeros(2, 2, 64), torch.zeros(2, 2, 64))


def test_operand_refusals():
    w = cca.MXTensor(*_held((2, 4), 64), "mxfp4", 64)
    with pytest.raises(ValueError):
        cca.mx.quantise(torch.zeros(3, 64), "int4")
    with pytest.raises(ValueError):
        cca.mx.quantise(torch.zeros(3, 64, dtype=torch.float64))
    with pytest.raises(ValueError):
        cca.mx.quantise(torch.zeros(3, 0))
    for x in (torch.zeros(2, 3, 32), torch.zeros(3, 64), torch.zeros(1, 3, 64)):
        with pytest.raises(ValueError):
            cca.mx.project(x, w)
    with pytest.raises(ValueError):
        cca.mx.project(torch.zeros(2, 3, 64), cca.MXTensor(*_held((2, 4), 64, "mxfp8"), "mxfp8", 64))


def test_cache_refusals():
    with pytest.raises(ValueError):
        cca.MXActivationCache(*_held((2, 3, 8), 64), "mxfp4", 64)
    cache = cca.MXActivationCache.empty(2, 8, 64, "mxfp4", device="cpu")
    for rows in ([0, 8], [-1], slice(4, 9), range(-1, 2)):
        with pytest.raises(IndexError):
            cache._resolve(rows)
    for rows in ([0.5], [[0, 1]], slice(0, 8, 2), range(0, 8, 2)):
        with pytest.raises(ValueError):
            cache._resolve(rows)
    assert cache._resolve(slice(None))[1:] == (0, 8) and cache._resolve(range(3, 3))[2] == 0 and cache._resolve([])[2] == 0


def test_library_refuses_before_it_launches():
    lib = nat.load()
    p = 4096                                            # an address nothing is launched on
    q = lambda *a: lib.clt_mx_quantise(*a)              # noqa: E731
    assert q(p, 4, 64, 64, 7, 0, p, p, None) == -2
    assert q(p, 4, 64, 64, 0, 3, p, p, None) == -1
    assert q(None, 4, 64, 64, 0, 0, p, p, None) == -1
    assert q(p, 4, 64, 63, 0, 0, p, p, None) == -1
    assert q(p, 4, 64, 64, 0, 0, p + 4, p, None) == -5
    assert q(p, 4, 262145, 262145, 0, 0, p, p, None) == -6
    assert q(p, -1, 64, 64, 0, 0, p, p, None) == -1
    assert q(None, 0, 64, 64, 0, 0, None, None, None) == 0
    w = lib.clt_mx_cache_write
    assert w(p, p, 256, 64, 0, None, 0, 6, 4, 64, 1, 0, p, p, 8, None, None) == -1      # past the last row
    assert w(p, p, 256, 64, 0, p, 16, 0, 4, 64, 1, 0, p, p, 8, p, None) == -1           # width of the row numbers
    assert w(p, p, 256, 64, 0, p, 32, 0, 4, 64, 1, 0, p, p, 8, None, None) == -1        # no scratch
    r = lib.clt_mx_cache_read
    assert r(p, p, 8, 0, None, 0, 5, 4, 64, 1, 0, None, None, None, None, 1.0, p, p, 0, 4, 0, None) == -1
    assert r(p, p, 8, 0, None, 0, 0, 4, 64, 1, 3, None, None, None, None, 1.0, p, p, 0, 4, 0, None) == -1
    assert r(p, p, 8, 0, None, 0, 0, 4, 64, 1, 0, None, None, None, None, 1.0, p, p, 1, 4, 0, None) == -1
    assert r(p, p, 0, 0, p, 32, 0, 4, 64, 1, 0, None, None, None, None, 1.0, p, p, 0, 4, 0, None) == -1
    e = lib.clt_mx_encode
    ws = lib.clt_mx_encode_workspace_bytes(400, 64, 512, 1, 0)
    assert ws >= 400 * 34 and lib.clt_mx_encode_workspace_bytes(4, 64, 16, 1, 1) == 0
    assert lib.clt_mx_encode_workspace_bytes(0, 64, 16, 1, 0) == 0 and lib.clt_mx_encode_workspace_bytes(4, 262145, 16, 1, 0) == 0
    assert e(p, None, p, p, None, p, 4, 64, 16, 1, 256, 0, 64, 15, 0, p, ws, None) == -1
    assert e(p, None, p, p, None, p, 4, 64, 16, 1, 256, 0, 64, 16, 5, p, ws, None) == -2
    assert e(p, None, p, p, None, p, 400, 64, 512, 1, 25600, 0, 204800, 512, 0, p, ws - 1, None) == -3
    assert e(p, None, p, p, None, p, 400, 64, 512, 1, 25600, 0, 204800, 512, 0, None, ws, None) == -3
    assert e(p, None, p + 8, p, None, p, 4, 64, 16, 1, 256, 0, 64, 16, 0, p, ws, None) == -5
    assert e(None, None, None, None, None, None, 0, 64, 16, 1, 0, 0, 64, 16, 0, None, 0, None) == 0
    assert e(p, None, p, p, None, p, 2 ** 20 + 1, 64, 16, 1, 256, 0, 64, 16, 0, p, ws, None) == -6
    f = lib.clt_mx_refresh
    assert f(p, 1, 4, 64, 256, 7, p, p, p, p, 0, None) == -2
    assert f(p, 1, 4, 64, 256, 0, p, p, None, p, 0, None) == -1
    assert f(p, 1, 4, 64, 256, 0, p, p, p + 64, p, 0, None) == -5
    assert f(p, 1, 0, 64, 256, 0, None, None, None, None, 0, None) == 0


def test_the_reciprocal_that_places_pieces_is_exact():
    """Rows of up to 2^16 pieces, counts up to pieces + 255: floor(at * ceil(2^32 / pieces) / 2^32) errs first at a multiple less one."""
    pieces = torch.arange(2, 65537, dtype=torch.int64)
    magic = (2 ** 32 + pieces - 1) // pieces
    for k in range(1, 130):
        at = k * pieces - 1
        ok = at > pieces + 254
        assert bool((ok | ((at * magic) >> 32 == at // pieces)).all())


def test_tile_kernels_spill_nothing(tmp_path):
    """The tiles' accumulators and fragments fill the 256 registers of two wavefronts per SIMD: one too many would go through
    memory in every stage while each result stays right.  Checked on the assembly the compiler
    reports for gfx950."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    out = tmp_path / "mx.s"
    flags = [f for f in clt_build.HIP_FLAGS if f != "-fPIC"]
    proc = subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", "-o", str(out), os.path.join(clt_build.CSRC, "mx.hip")],
                          stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert proc.returncode == 0, proc.stdout[-2000:]
    current, scratch = None, {}
    for line in open(out):
        m = re.match(r"^(_Z\w+):", line)
        if m:
            current = m.group(1)
        m = re.match(r"^; ScratchSize: (\d+)", line)
        if m and current:
            scratch[current] = int(m.group(1))
    tiles = {k: v for k, v in scratch.items() if "k_mx_project_tiles" in k}
    assert len(tiles) == 6, sorted(scratch)
    assert not any(tiles.values()), tiles
