"""Microscaled formats: cases that can be timed and compared with elementary torch operations.

A block of 32 neighbouring elements of a row shares one power of two; the elements are stored in 4 or 8 bits.

    block scale   byte s stands for 2^(s - 127), 255 for "no number"; s = exponent of the block's largest magnitude
                  minus the largest exponent of the element type, held in 0 .. 254; a block with an infinity or a NaN
                  gets 255 and reads back as NaN
    mxfp4         sign, 2 bits of exponent, 1 of mantissa: 0 0.5 1 1.5 2 3 4 6; two to a byte, the even one low
    mxfp8         sign, 4 bits of exponent, 3 of mantissa, up to 448
    mxint8        two's complement in 64ths, -127/64 .. 127/64
    rounding      to nearest, ties to even, beyond the largest value to the largest value

The operators:

    quantise      rows [n, d] to codes and scales, and the values they stand for
    write, read   a resident cache of activations [L, 2, rows, d] (inputs and targets of every layer): rows are
                  quantised as they are written, and gathered, expanded and normalised as they are read
    project       pre-activations x @ W.T + b of all layers at once: W in mxfp4, x quantised on the way in

Keys of a case
    op       "quantise", "write", "read" or "project"
    L, d     layers, elements of a row
    n        rows of a batch (tokens); R: rows that the cache holds; F: features per layer
    fmt      format of the codes
    dtype    type of the batch, of the biases and of the pre-activations
    norm     "none", "mean_std" or "sqrt_d_model" (read)
    rows     "run" (neighbouring rows of the cache) or "scattered" (write)
"""

import math

import torch

own = False

BLOCK = 32
EMAX = {"mxfp4": 2, "mxfp8": 8, "mxint8": 0}


def _case(name, op, L, d, n, fmt="mxfp4", dtype="bfloat16", F=0, R=0, norm="none", rows="scattered"):
    case = {"op": op, "L": L, "d": d, "n": n, "F": F, "R": R, "fmt": fmt, "dtype": dtype, "norm": norm, "rows": rows}
    return dict(case, name=name) if name else case


def listed():
    return [
        # encoder weights of the headline transcoder, quantised once when a model is made ready for serving
        _case("quantise_weights", "quantise", 12, 768, 24576),
        # rows of an odd width: one layer's activations of a small model, kept beside an analysis
        _case("quantise_ragged", "quantise", 1, 100, 333, "mxint8", "float16"),
        # a harvest step: the activations of one batch go to the next free rows of the cache
        _case("write_harvest", "write", 12, 768, 4096, "mxfp8", R=32768, rows="run"),
        # a shuffling buffer: the rows that the last batch used up are replaced, wherever they lie
        _case("write_scattered", "write", 24, 1024, 501, "mxfp4", R=8192),
        # a training batch drawn at random from the cache, normalised by the store's statistics
        _case("read_batch", "read", 12, 768, 4096, "mxfp8", R=32768, norm="mean_std"),
        # the same from 4-bit rows for a wide model kept in float32
        _case("read_wide", "read", 16, 2048, 3001, "mxfp4", "float32", R=16384, norm="sqrt_d_model"),
        # a few rows looked up for a dashboard
        _case("read_few", "read", 12, 640, 32, "mxint8", R=4096),
        # one token: interactive attribution, where the weights' one pass through the chip is the work
        _case("project_token", "project", 12, 768, 1, F=24576),
        # a short prompt
        _case("project_prompt", "project", 12, 768, 77, F=24576),
        # float32 outputs of a model whose widths and batch are no whole number of anything
        _case("project_ragged", "project", 6, 640, 301, dtype="float32", F=10006),
        # the headline batch
        _case("project_c1", "project", 12, 768, 4096, F=24576),
        # the widest rows: the products outweigh what is stored
        _case("project_wide", "project", 16, 2048, 8192, F=16384),
    ]


def _log_between(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["quantise", "write", "read", "project", "project", "project"])
    d = rng.choice([256, 512, 640, 768, 1024, 2048, 32 * rng.randint(1, 64), rng.randint(17, 2048)])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    L = rng.randint(1, 24)
    fmt = rng.choice(["mxfp4", "mxfp8", "mxint8"])
    if op == "project":
        F, n = _log_between(rng, 128, 32768), _log_between(rng, 1, 8192)
        F -= rng.choice([0, F % 8, F % 256 if F >= 256 else 0])
        while L * n * F * (d + 512) > 16 * 8192 * 16384 * 2560 or L * n * F * (2 if dtype == "float32" else 1) > 16 * 8192 * 16384:
            n = (n + 1) // 2
        return _case(None, op, L, d, n, "mxfp4", dtype, F=F)
    if op == "quantise":
        return _case(None, op, L, d, _log_between(rng, 1, 8192), fmt, dtype)
    R = _log_between(rng, 64, 16384)
    n = _log_between(rng, 1, min(R, 8192))
    norm = rng.choice(["none", "mean_std", "sqrt_d_model"]) if op == "read" else "none"
    return _case(None, op, L, d, n, fmt, dtype, R=R, norm=norm, rows=rng.choice(["run", "scattered"]) if op == "write" else "scattered")


# ---- the formats in elementary operations ------------------------------------------------------------------------

def _power(byte):
    """2^(byte - 127) as float32, from its bits; 255 is NaN."""
    b = byte.to(torch.int32)
    bits = torch.where(b == 0, torch.full_like(b, 0x00400000), torch.where(b == 255, torch.full_like(b, 0x7FC00000), b << 23))
    return bits.view(torch.float32)


def _blocks(x):
    """float32 [..., blocks, 32], the last block filled up with zeros."""
    d = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -d % BLOCK))
    return x.reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)


def _quantise(x, fmt):
    """(scale bytes [..., blocks], element values before scaling, float32 [..., blocks, 32])."""
    v = _blocks(x)
    expo = v.abs().amax(-1).view(torch.int32) >> 23
    byte = torch.where(expo == 255, expo, (expo - EMAX[fmt]).clamp(0, 254))
    v = v * _power(torch.where(expo == 255, expo, 254 - byte)).unsqueeze(-1)
    if fmt == "mxint8":
        return byte.to(torch.uint8), torch.round(v * 64).clamp(-127, 127) / 64
    if fmt == "mxfp8":
        return byte.to(torch.uint8), v.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    m = v.abs()
    q = (0.5 * ((m > 0.25).float() + (m >= 0.75).float() + (m > 1.25).float() + (m >= 1.75).float())
         + (m > 2.5).float() + (m >= 3.5).float() + 2.0 * (m > 5.0).float())
    return byte.to(torch.uint8), torch.where(m.isnan(), m, torch.copysign(q, v))


def _round_trip(x, fmt):
    """The values, float32 [..., d], that the codes of x stand for."""
    byte, q = _quantise(x, fmt)
    return (q * _power(byte).unsqueeze(-1)).flatten(-2)[..., :x.shape[-1]]


def _codes(x, fmt):
    """(codes uint8 [..., blocks * 16 or 32], scales uint8 [..., blocks]) as they are stored."""
    byte, q = _quantise(x, fmt)
    q = q.flatten(-2)
    if fmt == "mxint8":
        return (q * 64).to(torch.int8).view(torch.uint8), byte
    if fmt == "mxfp8":
        return q.to(torch.float8_e4m3fn).view(torch.uint8), byte
    m = q.abs()
    step = torch.where(m <= 2, 2 * m, torch.where(m == 6, m + 1, m + 2)).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
    return step[..., 0::2] | (step[..., 1::2] << 4), byte


def _expand(codes, scales, fmt, d):
    """float32 [..., d] of stored codes."""
    if fmt == "mxint8":
        q = codes.view(torch.int8).float() / 64
    elif fmt == "mxfp8":
        q = codes.view(torch.float8_e4m3fn).float()
    else:
        c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).to(torch.int32)
        m = c & 7
        m = torch.where(m <= 4, m * 0.5, torch.where(m == 7, torch.full_like(m, 6), m - 2).float())
        q = torch.where(c >= 8, -m, m)
    q = q.reshape(*q.shape[:-1], q.shape[-1] // BLOCK, BLOCK) * _power(scales).unsqueeze(-1)
    return q.flatten(-2)[..., :d]


# ---- inputs ------------------------------------------------------------------------------------------------------

def _activations(g, n, d, dtype):
    """Activations of one layer as language models have them: a scale per coordinate, a few outlying coordinates."""
    scale = torch.exp(0.5 * torch.randn(d, generator=g, device=g.device))
    scale[torch.randint(0, d, (4,), generator=g, device=g.device)] *= 20.0
    x = torch.randn(n, d, generator=g, device=g.device) * scale
    return (x / scale.square().mean().sqrt()).to(dtype)


class _State:
    pass


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    L, d, n, F, R, fmt = case["L"], case["d"], case["n"], case["F"], case["R"], case["fmt"]
    dtype = getattr(torch, case["dtype"])
    s = _State()
    s.case, s.dtype = case, dtype
    if case["op"] == "quantise":
        # weights of L layers, n rows each, or activations where there is one layer
        s.x = (((torch.rand(L, n, d, generator=g, device=dev) * 2 - 1) / math.sqrt(d)).to(dtype) if L > 1
               else _activations(g, n, d, dtype).unsqueeze(0))
        return s
    if case["op"] == "project":
        s.x = torch.stack([_activations(g, n, d, dtype) for _ in range(L)])
        pairs = [_codes((torch.rand(F, d, generator=g, device=dev) * 2 - 1) / math.sqrt(d), "mxfp4") for _ in range(L)]
        s.codes, s.scales = torch.stack([p[0] for p in pairs]), torch.stack([p[1] for p in pairs])
        s.bias = (0.1 * torch.randn(L, F, generator=g, device=dev)).to(dtype)
        return s
    blocks = -(-d // BLOCK)
    pitch = blocks * (16 if fmt == "mxfp4" else 32)
    s.codes = torch.zeros(L, 2, R, pitch, dtype=torch.uint8, device=dev)
    s.scales = torch.zeros(L, 2, R, blocks, dtype=torch.uint8, device=dev)
    if case["op"] == "write":
        s.x, s.tg = (torch.stack([_activations(g, n, d, dtype) for _ in range(L)]) for _ in range(2))
        if case["rows"] == "run":
            first = int(seed) % (R - n + 1)
            s.rows = slice(first, first + n)
        else:
            s.rows = torch.randperm(R, generator=g, device=dev)[:n]
        return s
    for l in range(L):
        for kind in range(2):
            s.codes[l, kind], s.scales[l, kind] = _codes(_activations(g, R, d, torch.float32), fmt)
    s.rows = torch.randint(0, R, (n,), generator=g, device=dev)     # a sampler's batch: any order, a row may come twice
    s.tables = None
    if case["norm"] == "mean_std":
        s.tables = tuple(t for _ in range(2) for t in (0.2 * torch.randn(L, d, generator=g, device=dev),
                                                       torch.rand(L, d, generator=g, device=dev) + 0.5))
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def _run_own(s):
    import crosslayer_coding_amd as cca

    case, op = s.case, s.case["op"]
    if op == "quantise":
        return cca.mx.quantise(s.x, case["fmt"]).dequantise(s.dtype)
    if op == "project":
        return cca.mx.project(s.x, cca.MXTensor(s.codes, s.scales, "mxfp4", case["d"]), s.bias)
    cache = cca.MXActivationCache(s.codes, s.scales, case["fmt"], case["d"])
    if op == "write":
        cache.write(s.rows, s.x, s.tg)
        return cache.read(s.rows, s.dtype)
    return cache.read(s.rows, s.dtype, case["norm"], s.tables)


def run(state):
    s, op = state, state.case["op"]
    if own:
        return _run_own(s)
    fmt, d = s.case["fmt"], s.case["d"]
    if op == "quantise":
        return _round_trip(s.x, fmt).to(s.dtype)
    if op == "write":
        return _round_trip(s.x, fmt).to(s.dtype), _round_trip(s.tg, fmt).to(s.dtype)
    if op == "project":
        w = _expand(s.codes, s.scales, "mxfp4", d)
        pre = torch.matmul(_round_trip(s.x, "mxfp4"), w.transpose(1, 2).contiguous())
        return (pre + s.bias.float().unsqueeze(1)).to(s.dtype)
    y = _expand(s.codes[:, :, s.rows], s.scales[:, :, s.rows], fmt, d)
    if s.tables is not None:
        mean = torch.stack((s.tables[0], s.tables[2]), dim=1).unsqueeze(2)
        y = (y - mean) / torch.stack((s.tables[1], s.tables[3]), dim=1).unsqueeze(2)
    elif s.case["norm"] == "sqrt_d_model":
        y = y * math.sqrt(d)
    y = y.to(s.dtype)
    return y[:, 0], y[:, 1]


def work(case):
    """Bytes and operations of one pass, every input, code and output counted once for each time that a pass needs it."""
    L, d, n, F = case["L"], case["d"], case["n"], case["F"]
    e = 4 if case["dtype"] == "float32" else 2
    row = -(-d // BLOCK) * (17 if case["fmt"] == "mxfp4" else 33)     # codes and scales of one row
    if case["op"] == "quantise":
        return {"bytes": L * n * (2.0 * d * e + 2 * row), "flops": 2.0 * L * n * d}     # read, stored; read back, given out
    if case["op"] == "write":
        return {"bytes": 2.0 * L * n * (2.0 * d * e + 2 * row), "flops": 4.0 * L * n * d}
    if case["op"] == "read":
        return {"bytes": 2.0 * L * n * (row + d * e) + 8 * n + (16.0 * L * d if case["norm"] == "mean_std" else 0), "flops": 4.0 * L * n * d}
    return {"bytes": L * (n * d * e + F * (row + e) + float(n) * F * e), "flops": 2.0 * L * n * F * d}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

_GRID4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _values64(x, fmt):
    """What the codes of x stand for: the format's definition, value by value, in float64."""
    d = x.shape[-1]
    v = torch.nn.functional.pad(x.double(), (0, -d % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = torch.frexp(v.abs().amax(-1, keepdim=True))[1] - 1                # floor(log2(largest)); 0 of a block of zeros
    scale = torch.pow(2.0, (top - EMAX[fmt]).clamp(min=-127).double())
    v = v / scale
    m, sign = v.abs(), torch.sign(v)
    if fmt == "mxint8":
        q = torch.clamp(torch.round(m * 64), max=127) / 64
    elif fmt == "mxfp8":
        quantum = torch.pow(2.0, ((torch.frexp(m)[1] - 1).clamp(min=-6) - 3).double())
        q = torch.clamp(torch.round(m / quantum) * quantum, max=448.0)
    else:
        grid = torch.tensor(_GRID4, dtype=torch.float64, device=x.device)
        half = (grid[1:] + grid[:-1]) / 2
        down, up = torch.searchsorted(half, m, right=False), torch.searchsorted(half, m, right=True)
        q = grid[torch.where(down % 2 == 0, down, up)]                     # they differ at a tie alone: the even code
    return (sign * q * scale).flatten(-2)[..., :d]


def _stored64(codes, scales, fmt, d):
    c = codes.to(torch.int64)
    if fmt == "mxint8":
        q = torch.where(c >= 128, c - 256, c).double() / 64
    elif fmt == "mxfp8":
        e, m = (c >> 3) & 15, (c & 7).double()
        q = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.pow(2.0, (e - 10).double())) * torch.where(c >= 128, -1.0, 1.0)
    else:
        c = torch.stack((c % 16, c // 16), dim=-1).flatten(-2)
        q = torch.tensor(_GRID4 + tuple(-v for v in _GRID4), dtype=torch.float64, device=c.device)[c]
    return (q.unflatten(-1, (-1, BLOCK)) * torch.pow(2.0, scales.double() - 127).unsqueeze(-1)).flatten(-2)[..., :d]


def exact(case, seed):
    s = prepare(case, seed)
    L, d, n, F, fmt = case["L"], case["d"], case["n"], case["F"], case["fmt"]
    if case["op"] == "quantise":
        return torch.stack([_values64(s.x[l], fmt) for l in range(L)])
    if case["op"] == "write":
        return tuple(torch.stack([_values64(v[l], fmt) for l in range(L)]) for v in (s.x, s.tg))
    if case["op"] == "project":
        pre = torch.empty(L, n, F, dtype=torch.float64, device=s.x.device)
        for l in range(L):
            pre[l] = _values64(s.x[l], "mxfp4") @ _stored64(s.codes[l], s.scales[l], "mxfp4", d).t() + s.bias[l].double()
        return pre
    out = []
    for kind in range(2):
        y = torch.stack([_stored64(s.codes[l, kind][s.rows], s.scales[l, kind][s.rows], fmt, d) for l in range(L)])
        if case["norm"] == "mean_std":
            y = (y - s.tables[2 * kind].double().unsqueeze(1)) / s.tables[2 * kind + 1].double().unsqueeze(1)
        elif case["norm"] == "sqrt_d_model":
            y = y * math.sqrt(d)
        out.append(y)
    return tuple(out)
