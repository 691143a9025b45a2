"""spmm24_quantize_int8 and spmm24_launch_int8 against the plain formulas in
64 bits.  Quantised values are compared bit for bit; products within the
rounding bound that int8_problems.tolerance derives."""
import numpy as np
import pytest

import spmm24
from int8_problems import act64, bits_to_f64, problem, product, prune_int8, round_bits, tolerance

pytestmark = pytest.mark.gpu


def _dev(a, device):
    import torch

    a = np.ascontiguousarray(a)
    if a.dtype == np.uint16:
        a = a.view(np.int16)
    return torch.from_numpy(a.copy()).to(device)


# ------------------------------------------------------------- quantise
def _quantized(x64):
    """(q, scale) of float64 rows, by the formula."""
    a = np.abs(x64).max(1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where((a > 0) & np.isfinite(a), np.rint(127 * x64 / a), 0)
    q[~np.isfinite(q)] = 0
    with np.errstate(over="ignore"):
        return q.astype(np.int8), (a[:, 0] / 127).astype(np.float32)


def _check_quantize(device, bits, bf16, packed=False, ld=0, offset=0):
    import torch

    rows, cols = bits.shape
    if packed:
        pad = np.full(((rows + 7) // 8 * 8, cols), 0x7E00 if not bf16 else 0x7FC0, dtype=np.uint16)  # NaN pad rows
        pad[:rows] = bits
        host = pad.reshape(-1, 8, cols).transpose(0, 2, 1).reshape(-1)
    else:
        step = ld or cols
        host = np.full(offset + rows * step, 0x7C00, dtype=np.uint16)  # what lies between rows is not read
        for r in range(rows):
            host[offset + r * step: offset + r * step + cols] = bits[r]
    x = _dev(host, device)[offset:]
    guard = 64
    qbuf = torch.full((rows * cols + guard,), 77, dtype=torch.int8, device=device)
    sbuf = torch.full((rows + guard,), -3.0, device=device)
    q, s = spmm24.quantize_int8(x, rows, cols, qbuf, sbuf, bf16=bf16, packed=packed, ld=ld)
    torch.cuda.synchronize(device)
    want_q, want_s = _quantized(bits_to_f64(bits, bf16).reshape(rows, cols))
    got_q = q.cpu().numpy()
    assert (got_q[rows * cols:] == 77).all() and (s[rows:] == -3.0).all(), "wrote behind the last row"
    assert np.array_equal(got_q[: rows * cols].reshape(rows, cols), want_q)
    assert np.array_equal(s[:rows].cpu().numpy(), want_s, equal_nan=True)


def _random_bits(rows, cols, bf16, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * np.exp(2 * rng.standard_normal((rows, 1)))
    return round_bits(x.astype(np.float32), bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 8), (9, 31), (5, 256), (1, 1000), (130, 4096), (7, 11008),
                                       (2, 40000), (3, 40001), (2, 70008), (1, 70001)])
def test_quantize_rows(cuda_device, rows, cols, bf16):
    _check_quantize(cuda_device, _random_bits(rows, cols, bf16, rows + cols), bf16)


@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 8), (8, 64), (9, 256), (3, 4096), (17, 4104), (33, 11008), (9, 40008),
                                       (1300, 264)])
def test_quantize_strips(cuda_device, rows, cols, bf16):
    _check_quantize(cuda_device, _random_bits(rows, cols, bf16, rows + cols), bf16, packed=True)


@pytest.mark.parametrize("ld,offset", [(264, 0), (261, 0), (256, 3), (300, 8)])
def test_quantize_strides_and_alignment(cuda_device, ld, offset):
    _check_quantize(cuda_device, _random_bits(5, 256, False, ld), False, ld=ld, offset=offset)


def _all_below(top, bf16):
    """Every finite value of the type with magnitude at most `top` (bits), both signs."""
    pos = np.arange(top + 1, dtype=np.uint16)
    return np.concatenate([pos, pos | 0x8000, [top]]).astype(np.uint16)


@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
def test_quantize_rounds_every_value_exactly(cuda_device, bf16):
    """All values below maxima of every size: the smallest subnormals, the
    largest finite value, powers of two, 127 2^e (whose halves are ties), odd
    significands."""
    one = 0x3F80 if bf16 else 0x3C00
    last = 0x7F7F if bf16 else 0x7BFF
    ties = [int(round_bits(np.float32(127.0 * 2.0 ** e), bf16)) for e in (-20, -7, -1, 0, 3, 8)]
    tops = [1, 2, 3, 127, 128, 129, one - 1, one, one + 1, last, last - 1] + ties
    tops += [int(t) for t in np.random.default_rng(3).integers(4, last, 12)]
    for packed in (False, True):
        for top in tops:
            row = _all_below(top, bf16)
            cols = (len(row) + 7) // 8 * 8
            bits = np.zeros((1, cols), dtype=np.uint16)
            bits[0, : len(row)] = row
            _check_quantize(cuda_device, bits, bf16, packed=packed)


@pytest.mark.parametrize("packed", [False, True], ids=["rows", "strips"])
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
def test_quantize_zeros_infinities_and_nan(cuda_device, bf16, packed):
    inf = 0x7F80 if bf16 else 0x7C00
    bits = _random_bits(7, 128, bf16, 5)
    bits[0] = 0
    bits[1] = 0x8000
    bits[2, 5] = inf
    bits[3, 127] = inf | 0x8000
    bits[4, 0] = inf + 1  # NaN
    bits[5, 3], bits[5, 4] = inf, inf | 0x8041
    _check_quantize(cuda_device, bits, bf16, packed=packed)


# -------------------------------------------------------------- product
def _run(device, M, N, K, *, split=0, bf16=False, w=True, xs=True, bias=False, residual=False, inplace=False, alpha=1.0,
         act=0, packed=False, seed=0, flags=0, stream=None, ab=None):
    import torch

    a, b = ab or problem(M, N, K, seed)
    vals, meta = spmm24.compress_a_int8(a, M, K)
    rng = np.random.default_rng(seed + 7)
    acc = product(a, b)
    size = np.sqrt(K) * 4000.0
    w_scale = (rng.uniform(0.5, 2.0, M) / size).astype(np.float32) if w else None
    x_scale = rng.uniform(0.25, 4.0, N).astype(np.float32) if xs else None
    if not w:
        alpha = alpha / size
    bias_bits = round_bits(rng.standard_normal(M), bf16) if bias else None
    res_bits = round_bits(rng.standard_normal((M, N)), bf16) if residual else None
    strips = (N + 7) // 8

    def layout(m):
        if not packed:
            return m.reshape(-1)
        pad = np.zeros((M, strips * 8), dtype=np.uint16)
        pad[:, :N] = m
        return pad.reshape(M, strips, 8).transpose(1, 0, 2).reshape(-1)

    n_out = strips * 8 * M if packed else M * N
    guard = 128
    c = torch.full((n_out + guard,), -1, dtype=torch.int16, device=device)
    res_dev = None
    if residual:
        if inplace:
            c[:n_out] = _dev(layout(res_bits), device)
            res_dev = c
        else:
            res_dev = _dev(layout(res_bits), device)
    args = dict(w_scale=None if w_scale is None else _dev(w_scale, device),
                x_scale=None if x_scale is None else _dev(x_scale, device),
                bias=None if bias_bits is None else _dev(bias_bits, device), residual=res_dev)
    dv, db, dm = _dev(vals, device), _dev(b, device), _dev(meta, device)
    torch.cuda.synchronize(device)
    rc = spmm24.launch_int8(stream, dv, db, dm, c, M, N, K, split_k=split, flags=flags | (spmm24.BF16 if bf16 else 0),
                            alpha=alpha, activation=act,
                            out_layout=spmm24.OUT_PACKED_B if packed else spmm24.OUT_ROW_MAJOR, **args)
    assert rc == 0, spmm24._lib.spmm24_last_error().decode()
    torch.cuda.synchronize(device)
    assert spmm24.device_status(device.index or 0) == 0
    bits = c.cpu().numpy().view(np.uint16)
    assert (bits[n_out:] == 0xFFFF).all(), "wrote behind C"
    bits = bits[:n_out]
    if packed:
        full = bits.reshape(strips, M, 8).transpose(1, 0, 2).reshape(M, strips * 8)
        assert not full[:, N:].any(), "pad columns of a packed C must be zero"
        bits = full[:, :N]
    bits = np.ascontiguousarray(bits.reshape(M, N))
    pre = np.float64(np.float32(alpha)) * acc
    if w:
        pre = pre * w_scale.astype(np.float64)[:, None]
    if xs:
        pre = pre * x_scale.astype(np.float64)
    base = np.zeros((M, 1))
    if bias:
        base = bits_to_f64(bias_bits, bf16).reshape(M, 1)
    extra = bits_to_f64(res_bits, bf16).reshape(M, N) if residual else 0.0
    ref = act64(pre + base, act) + extra
    got = bits_to_f64(bits, bf16).reshape(M, N)
    tol = tolerance(ref, np.abs(pre) + np.abs(base), extra, act, bf16)
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(np.abs(got - ref) / tol)))
    return bits


# every N tile of the cluster kernel, K splits, an odd number of 128-K groups
# (half-filled last stage), ragged M and N, one token; then the pair kernels
SHAPES = [(128, 16, 128, 0), (16, 1, 128, 0), (256, 16, 384, 0), (4096, 1, 4096, 0), (4096, 13, 11008, 0),
          (2048, 32, 2048, 3), (1024, 64, 1024, 0), (144, 33, 640, 0), (512, 128, 512, 0), (256, 200, 768, 0),
          (256, 300, 768, 0), (384, 24, 1152, 8), (1040, 509, 1024, 0), (2048, 2047, 768, 0), (512, 512, 12800, 0)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_int8_matches_the_formula(cuda_device, shape):
    M, N, K, split = shape
    _run(cuda_device, M, N, K, split=split, seed=M + N + K)


@pytest.mark.parametrize("shape", [(256, 5, 512), (272, 48, 640), (512, 320, 768), (2064, 2041, 512)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("act", [0, 1, 2, 3], ids=["none", "relu", "silu", "gelu"])
def test_int8_epilogues(cuda_device, shape, bf16, act):
    M, N, K = shape
    _run(cuda_device, M, N, K, bf16=bf16, bias=True, act=act, seed=act)
    _run(cuda_device, M, N, K, bf16=bf16, bias=True, residual=True, act=act, alpha=0.7, seed=act + 9)
    _run(cuda_device, M, N, K, bf16=bf16, residual=True, inplace=True, packed=True, act=act, seed=act + 19)
    _run(cuda_device, M, N, K, bf16=bf16, packed=True, act=act, w=False, xs=act == 0, seed=act + 29)


@pytest.mark.parametrize("kw", [dict(pair=1, pair2=0, pair_split=1), dict(pair=1, pair2=0, pair_split=2),
                                dict(pair=1, pair2=1), dict(pair=0, tile_n=256), dict(pair=0, tile_n=128),
                                dict(pair=0, tile_n=64, deep_ring=1), dict(pair=0, tile_n=32, deep_ring=1),
                                dict(pair=0, tile_n=16, deep_ring=1), dict(pair=0, tile_n=32), dict(pair=0, tile_n=16)],
                         ids=lambda k: "-".join("%s%s" % i for i in k.items()))
def test_every_kernel_gives_the_same_bits(cuda_device, tuning, kw):
    """The sums are exact, so every kernel, tile and K split gives the same bits."""
    M, N, K = 528, 269, 1024
    tuning(pair=0)
    want = _run(cuda_device, M, N, K, split=1, bias=True, act=2, seed=3)
    tuning(**kw)
    assert np.array_equal(_run(cuda_device, M, N, K, bias=True, act=2, seed=3), want)


# more 512 x 224 tiles than pairs of SMs: the persistent kernel, two and three
# tiles a pair, one to five stages of K, ragged M and N
@pytest.mark.parametrize("M,N,K,kw", [
    (5120, 2048, 256, dict()), (5136, 2040, 512, dict(bf16=True, bias=True, act=2)),
    (5008, 2008, 768, dict(packed=True, act=1, bias=True)), (5120, 2041, 1024, dict(packed=True, bf16=True)),
    (11008, 2048, 1280, dict(alpha=0.5, act=3)), (5120, 2048, 512, dict(w=False, xs=False)),
    (4624, 2240, 512, dict(flags=spmm24.STATIC_WEIGHTS)),
], ids=lambda v: str(v) if isinstance(v, int) else "-".join(v))
def test_persistent_tiles(cuda_device, tuning, M, N, K, kw):
    tuning(pair2=1)
    got = _run(cuda_device, M, N, K, seed=K, **kw)
    tuning(pair2=0)  # the sums are exact: another kernel, the same bits
    assert np.array_equal(_run(cuda_device, M, N, K, seed=K, **kw), got)


def test_persistent_tiles_back_to_back(cuda_device):
    """Launches that overlap (each reads what the one before wrote), many tiles each."""
    import torch

    M, N, K = 5120, 2048, 512
    a, b = problem(M, N, K, 5)
    vals, meta = spmm24.compress_a_int8(a, M, K)
    dv, dm, db = _dev(vals, cuda_device), _dev(meta, cuda_device), _dev(b, cuda_device)
    st = torch.cuda.current_stream(cuda_device)
    scale = torch.ones(N, device=cuda_device)
    outs = [torch.zeros(M, N, dtype=torch.float16, device=cuda_device) for _ in range(6)]
    for i, c in enumerate(outs):
        scale.fill_(2.0 ** -(8 + i))
        assert spmm24.launch_int8(st, dv, db, dm, c, M, N, K, x_scale=scale, flags=spmm24.STATIC_WEIGHTS) == 0
    torch.cuda.synchronize()
    acc = torch.from_numpy(product(a, b)).to(cuda_device)
    for i, c in enumerate(outs):
        assert torch.equal(c, (acc * 2.0 ** -(8 + i)).to(torch.float32).to(torch.float16))
    assert spmm24.device_status(0) == 0


@pytest.mark.parametrize("split", range(1, 9))
def test_splits_give_the_same_bits(cuda_device, split):
    want = _run(cuda_device, 272, 21, 2176, split=1, seed=4)
    assert np.array_equal(_run(cuda_device, 272, 21, 2176, split=split, seed=4), want)


@pytest.mark.parametrize("sign", [1, -1])
def test_largest_sums_do_not_overflow(cuda_device, sign):
    """K = 262016: 131008 products of 2^14 each, 99.95 % of 2^31."""
    M, N, K = 16, 2, 262016
    a = np.zeros((M, K), dtype=np.int8)
    a[:, 0::4] = a[:, 2::4] = -128
    b = np.full((N, K), -128 if sign > 0 else 127, dtype=np.int8)
    _run(cuda_device, M, N, K, ab=(a, b), split=0)
    _run(cuda_device, M, N, K, ab=(a, b), split=1, bf16=True)


def test_infinite_scale_makes_its_token_nan(cuda_device):
    import torch

    M, K, N = 64, 256, 9
    a, _ = problem(M, 1, K, 1)
    x = np.random.default_rng(2).standard_normal((N, K)).astype(np.float16)
    x[4, 9] = np.inf
    x[6, 0] = np.nan
    q, s = spmm24.quantize_int8(torch.from_numpy(x).to(cuda_device), N, K)
    vals, meta = spmm24.compress_a_int8(a, M, K)
    c = torch.zeros(M, N, dtype=torch.float16, device=cuda_device)
    rc = spmm24.launch_int8(torch.cuda.current_stream(cuda_device), _dev(vals, cuda_device), q, _dev(meta, cuda_device),
                            c, M, N, K, x_scale=s, alpha=1e-3)
    assert rc == 0
    nan = torch.isnan(c).cpu().numpy()
    assert nan[:, [4, 6]].all() and not nan[:, [0, 1, 2, 3, 5, 7, 8]].any()


@pytest.mark.parametrize("M,K", [(16, 128), (272, 640)])
@pytest.mark.parametrize("prune", [False, True])
def test_device_packer_matches_the_host(cuda_device, M, K, prune):
    import torch

    a = np.random.default_rng(M).integers(-128, 128, (M, K)).astype(np.int8)
    a[0, :12] = [-128, 127, -127, 1, 5, -5, 5, -5, 0, -128, 0, 0]
    if not prune:
        a = prune_int8(a, M, K)
    want = spmm24.compress_a_int8(prune_int8(a, M, K), M, K)
    bad = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    vals, meta = spmm24.pack_a_int8_device(_dev(a, cuda_device), M, K, prune=prune, bad_blocks=bad)
    assert int(bad.item()) == 0
    assert np.array_equal(vals.cpu().numpy(), want[0]) and np.array_equal(meta.cpu().numpy(), want[1])
    if not prune:
        a[5, :3] = -128  # three values in a group
        spmm24.pack_a_int8_device(_dev(a, cuda_device), M, K, bad_blocks=bad)
        assert int(bad.item()) == 1


# ------------------------------------------------------ used together
def _mlp(device, T, H, inter, bf16, stream, steps=1, graph=False):
    """Weights pruned, quantised and packed on the device, then per step:
    quantise tokens, up projection with SiLU into strips, quantise the strips,
    down projection.  Returns what each call read and wrote."""
    import torch

    dt = torch.bfloat16 if bf16 else torch.float16
    g = torch.Generator(device=device).manual_seed(11)
    s = {}
    with torch.cuda.stream(stream):
        for name, (M, K) in {"up": (inter, H), "down": (H, inter)}.items():
            w = (torch.randn(M, K, generator=g, device=device) * 0.02).to(dt)
            spmm24.prune_2of4_device(w, M, K, bf16=bf16)
            q, scale = spmm24.quantize_int8(w, M, K, bf16=bf16)
            s[name] = (*spmm24.pack_a_int8_device(q, M, K), scale, q)
        x = torch.randn(T, H, generator=g, device=device).to(dt)
        strips = (T + 7) // 8
        s |= {"x": x, "q1": torch.empty(T, H, dtype=torch.int8, device=device), "s1": torch.empty(T, device=device),
              "h": torch.empty(strips, inter, 8, dtype=dt, device=device),
              "q2": torch.empty(T, inter, dtype=torch.int8, device=device), "s2": torch.empty(T, device=device),
              "y": torch.empty(H, T, dtype=dt, device=device)}

        def step():
            flags = spmm24.STATIC_WEIGHTS | (spmm24.BF16 if bf16 else 0)
            st = torch.cuda.current_stream(device)
            spmm24.quantize_int8(s["x"], T, H, s["q1"], s["s1"], bf16=bf16)
            up, down = s["up"], s["down"]
            assert spmm24.launch_int8(st, up[0], s["q1"], up[1], s["h"], inter, T, H, w_scale=up[2], x_scale=s["s1"],
                                      flags=flags, activation=spmm24.ACT_SILU, out_layout=spmm24.OUT_PACKED_B) == 0
            spmm24.quantize_int8(s["h"], T, inter, s["q2"], s["s2"], bf16=bf16, packed=True)
            assert spmm24.launch_int8(st, down[0], s["q2"], down[1], s["y"], H, T, inter, w_scale=down[2],
                                      x_scale=s["s2"], flags=flags) == 0

        stream.synchronize()
        if graph:
            step()
            stream.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=stream):
                step()
            for i in range(steps):
                s["x"].copy_(torch.roll(s["x"], 1, 1))
                gr.replay()
        else:
            for i in range(steps):
                step()
    torch.cuda.synchronize(device)
    return s


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("T,H,inter", [(1, 256, 640), (13, 512, 1408), (300, 384, 896)])
def test_mlp_of_two_layers(cuda_device, T, H, inter, bf16, graph):
    import torch

    s = _mlp(cuda_device, T, H, inter, bf16, torch.cuda.Stream(cuda_device), steps=3, graph=graph)
    n = lambda t: t.cpu().numpy()  # noqa: E731
    bits = lambda t: n(t.view(torch.int16)).view(np.uint16)  # noqa: E731
    q1, s1 = _quantized(bits_to_f64(bits(s["x"]), bf16).reshape(T, H))
    assert np.array_equal(n(s["q1"]), q1) and np.array_equal(n(s["s1"]), s1)
    pre = product(n(s["up"][3]), q1) * n(s["up"][2]).astype(np.float64)[:, None] * s1.astype(np.float64)
    ref = act64(pre, 2)
    h = bits_to_f64(bits(s["h"]), bf16).reshape(-1, inter, 8).transpose(1, 0, 2).reshape(inter, -1)
    assert (np.abs(h[:, :T] - ref) <= tolerance(ref, pre, 0.0, 2, bf16)).all() and not h[:, T:].any()
    q2, s2 = _quantized(np.ascontiguousarray(h[:, :T].T))
    assert np.array_equal(n(s["q2"]), q2) and np.array_equal(n(s["s2"]), s2)
    ref = product(n(s["down"][3]), q2) * n(s["down"][2]).astype(np.float64)[:, None] * s2.astype(np.float64)
    y = bits_to_f64(bits(s["y"]), bf16).reshape(H, T)
    assert (np.abs(y - ref) <= tolerance(ref, ref, 0.0, 0, bf16)).all()
