"""spmm24_launch_moe where its values are delicate: rows of h next to ties,
rows of tiny values, gates far below zero, epilogues of tokens that hold no
number, and 17 to 32 tokens with the experts in two groups."""
import numpy as np
import pytest

import spmm24
from act_values import act_tails
from test_gpu_moe import Layer, _matrix, _strips

pytestmark = pytest.mark.gpu


def _round_exactly(h, a):
    """rint(127 h / a), ties to even, of integers."""
    n, d = 127 * np.abs(h), a
    q, r = n // d, n % d
    q = q + ((2 * r > d) | ((2 * r == d) & (q % 2 == 1)))
    return np.sign(h) * q


def _hard_rows(count, seed):
    """Rows of 128 integers, the first the largest: values on a tie or next to one, those first that a product with
    the rounded quotient 127 / a takes to the wrong side."""
    rng = np.random.default_rng(seed)
    rows = []
    while len(rows) < count:
        a = int(rng.integers(100000, 400000))
        if len(rows) % 2:
            a = 254 * (a // 508 * 2 + 1)  # (2k + 1) a / 254 is an integer: exact ties
            a = a if a < 400000 else a - 254 * 400
        k = np.arange(127)
        h = np.concatenate([(2 * k + 1) * a // 254 + d for d in (0, 1)])
        h = np.concatenate([h, -h])
        h = h[(np.abs(h) <= a)]
        fast = np.rint(h.astype(np.float32) * (np.float32(127) / np.float32(a)))
        wrong = fast != _round_exactly(h, a)
        order = np.argsort(~wrong, kind="stable")
        rows.append(np.concatenate([[a], h[order][:127]]))
    rows = np.array(rows)
    fast = np.rint(rows.astype(np.float32) * (np.float32(127) / rows[:, :1].astype(np.float32)))
    assert (fast != _round_exactly(rows, rows[:, :1])).any()  # hard ones are among them
    return rows


def _integer_layer(device, rows, unit, d_scale):
    """T tokens, each with an expert of its own whose h is the integers `rows` times unit ** 2: gate rows that sum
    to them, up rows that pick a one, the identity for down."""
    import torch

    T, H = rows.shape[0], 128
    x = np.full(H, 127, dtype=np.float32)  # scale 1
    x[4] = 1
    gu = np.zeros((T, 2 * H, H), dtype=np.int8)
    for e in range(T):
        for i, v in enumerate(rows[e]):
            tens = int(np.round(v / 127))
            gu[e, i, 4] = v - 127 * tens
            for k in list(range(8, 128, 4)) + list(range(9, 128, 4)):  # at most two of each four
                w = int(np.clip(tens, -127, 127))
                gu[e, i, k] = w
                tens -= w
            assert tens == 0 and abs(v) < 127 * 127 * 60
            gu[e, H + i, 4] = 1
        assert np.array_equal(gu[e].astype(np.int64) @ x.astype(np.int64), np.concatenate([rows[e], np.ones(H, np.int64)]))
    eye = np.tile(np.eye(H, dtype=np.int8), (T, 1))
    up = lambda m: [torch.from_numpy(v).to(device) for v in spmm24.compress_a_int8(m, m.shape[0], H)]  # noqa: E731
    return (torch.from_numpy(x).to(device).expand(T, H), up(gu.reshape(-1, H)), up(eye),
            torch.full((T * 2 * H,), unit, device=device), torch.full((T * H,), d_scale, device=device))


@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("unit,d_scale", [(1.0, 1.0), (2.0 ** -70, 2.0 ** 120)], ids=["ones", "tiny"])
def test_rows_of_h_round_exactly(cuda_device, unit, d_scale, bf16):
    """Ties, their neighbours, and rows whose largest value is near the end of fp32's range (where 127 / max
    overflows): every int8 value of h is what the formula gives."""
    import torch

    T, H = 32, 128
    rows = _hard_rows(T, 1)
    dt = torch.bfloat16 if bf16 else torch.float16
    x, gu, dn, gs, ds = _integer_layer(cuda_device, rows, unit, d_scale)
    flags = spmm24.MOE_INT8 | (spmm24.BF16 if bf16 else 0)
    ws = torch.zeros(spmm24.moe_workspace_bytes(T, H, H, T, 1, flags), dtype=torch.uint8, device=cuda_device)
    ids = torch.arange(T, dtype=torch.int32, device=cuda_device).reshape(T, 1)
    w = 2.0 ** -8
    weights = torch.full((T, 1), w, device=cuda_device)
    y = torch.zeros(H, T, dtype=dt, device=cuda_device)
    rc = spmm24.launch_moe(torch.cuda.current_stream(cuda_device), _strips(x.to(dt)), None, gu[0], gu[1], dn[0], dn[1], y, T, H,
                           H, T, 1, ws, flags=flags, gate_up_scale=gs, down_scale=ds, topk_ids=ids, topk_weights=weights,
                           activation=spmm24.ACT_NONE)
    assert rc == 0, spmm24._lib.spmm24_last_error().decode()
    a = rows[:, 0].astype(np.float64) * unit * unit
    # y = w a / 127 d q, off by 2^-8 of 127 at most and a few fp32 steps (2^-20 for a / 127 next to fp32's smallest): below 1/2
    q = y.double().cpu().numpy().T / (w * a / 127 * d_scale)[:, None]
    assert np.array_equal(np.rint(q).astype(np.int64), _round_exactly(rows, rows[:, :1]))
    assert spmm24.device_status(0) == 0


@pytest.mark.parametrize("act", [2, 3], ids=["silu", "gelu"])
def test_gates_far_below_zero(cuda_device, act):
    """Gates down to where e^-gate overflows fp32, times an up value of 2^100 that makes the smallest products
    ordinary numbers: h is held to the activation's own size.

    Bound, relative: expf, 1 + e, the quotient, the products: 10 steps of 2^-23, and 16 more where e^x is below 2^-126
    (four bits are lost at e^-90); GELU's exponent is off by seven roundings of 2^-24, which e^x sees |x| times.  h and y
    round to bf16 once each."""
    import torch

    H = 128
    gates = np.linspace(-90, 8, H) if act == 2 else np.linspace(-10.1, 8, H)
    w = torch.zeros(2 * H, H, dtype=torch.bfloat16, device=cuda_device)
    w[:H, 0] = torch.from_numpy(gates).to(cuda_device).bfloat16()
    w[H:, 0] = 2.0 ** 100
    gate = w[:H, 0].double()
    x = torch.zeros(1, H, dtype=torch.bfloat16, device=cuda_device)
    x[0, 0] = 1
    gu = spmm24.pack_a_device(w, 2 * H, H)[:2]
    dn = spmm24.pack_a_device(torch.eye(H, dtype=torch.bfloat16, device=cuda_device), H, H)[:2]
    ws = torch.zeros(spmm24.moe_workspace_bytes(1, H, H, 1, 1, spmm24.BF16), dtype=torch.uint8, device=cuda_device)
    ids = torch.zeros(1, 1, dtype=torch.int32, device=cuda_device)
    y = torch.zeros(H, 1, dtype=torch.bfloat16, device=cuda_device)
    rc = spmm24.launch_moe(torch.cuda.current_stream(cuda_device), _strips(x), None, gu[0], gu[1], dn[0], dn[1], y, 1, H, H, 1, 1,
                           ws, flags=spmm24.BF16, topk_ids=ids, topk_weights=torch.ones(1, 1, device=cuda_device),
                           activation=act)
    assert rc == 0, spmm24._lib.spmm24_last_error().decode()
    ref, size = act_tails(gate, act)
    ref = ref * 2.0 ** 100
    rel = (26 + (0 if act == 2 else 3.5) * size) * 2.0 ** -23
    off = (y[:, 0].double() - ref).abs()
    tol = ref.abs() * (rel + 2 * 2.0 ** -8)
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("act", [1, 2, 3], ids=["relu", "silu", "gelu"])
@pytest.mark.parametrize("T", [3, 16, 20], ids=lambda t: "T%d" % t)
@pytest.mark.parametrize("int8", [False, True], ids=["fp16", "int8"])
def test_epilogue_activations(cuda_device, act, T, int8):
    """An activation of y: tokens with an infinity or NaN keep it, and values far below zero are right beside their
    own size (one expert of weight 1; alpha makes most of y lie in -12 .. 12)."""
    import torch

    L = Layer(cuda_device, 256, 384, 4, int8=int8, seed=act)
    x = L.tokens(T)
    x[1, 5] = float("nan")
    x[2, 9] = float("inf")
    ids = torch.randint(0, 4, (T, 1), generator=L.g, device=cuda_device, dtype=torch.int32)
    w = torch.ones(T, 1, device=cuda_device)
    ws = L.workspace(T, 1)
    pre, _, _ = L.run(x, 1, ws, ids=ids, weights=w)
    scale = 2.0 ** float(torch.log2(4 / L.result(pre, T)[:, 3 if T > 3 else 0].std()).round())
    bias = torch.zeros(256, dtype=torch.float16, device=cuda_device)
    bias[::2] = -6
    out, _, _ = L.run(x, 1, ws, ids=ids, weights=w, alpha=scale, bias=bias, epilogue_activation=act)
    got = L.result(out, T)
    assert torch.isnan(got[:, 1]).all() and not torch.isfinite(got[:, 2]).any()
    keep = [t for t in range(T) if t not in (1, 2)]
    # y before the activation, to 16 bits, from the layer itself; the activated one must come of a value that rounds to it
    lin, _, _ = L.run(x, 1, ws, ids=ids, weights=w, alpha=scale, bias=bias)
    lin = L.result(lin, T)[:, keep]
    got = got[:, keep]
    assert (lin < -7).any() and (lin > 0).any()
    step = 2.0 ** -11 * lin.abs() + 2.0 ** -25
    if act == 1:
        assert torch.equal(got, lin.clamp(min=0))
        return
    ref, size = act_tails(lin, act)
    lo, hi = act_tails(lin - step, act)[0], act_tails(lin + step, act)[0]
    spread = (lo - ref).abs().maximum((hi - ref).abs())
    rel = (5 + 4.7 * size.clamp(max=110)) * 2.0 ** -23
    off = (got - ref).abs()
    tol = spread + (ref.abs() + spread) * (2.0 ** -11 + 2 * rel) + 2.0 ** -25
    assert (off <= tol).all(), float((off / tol).max())


# hidden x inter so that gate / up has eight units or more for each CTA, and down a tile or less
TWO_GROUPS = [(17, 2048, 1152, 20, 4), (32, 4096, 1408, 8, 2), (19, 3200, 1408, 9, 3), (31, 2176, 2816, 16, 2)]


@pytest.mark.parametrize("shape", TWO_GROUPS, ids=lambda s: "T%d-%dx%d-E%dk%d" % s)
@pytest.mark.parametrize("kind", ["fp16", "bf16", "int8-fp16", "int8-bf16"])
def test_many_tokens_in_two_groups(cuda_device, shape, kind):
    import torch

    T, H, inter, E, k = shape
    int8 = kind.startswith("int8")
    L = Layer(cuda_device, H, inter, E, bf16=kind.endswith("bf16"), int8=int8, seed=T + E)
    x = L.tokens(T)
    ids, w, w_err = L.routed(x, k, True)
    sms = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    stages = (H // (128 if int8 else 64) + 1) // 2
    assert len(ids.unique()) * -(-inter // 128) * stages >= 8 * sms and -(-H // 128) <= sms  # two groups
    ws = L.workspace(T, k)
    out, got_ids, got_w = L.run(x, k, ws)
    got = L.result(out, T)
    assert torch.equal(got_ids.long(), ids) and ((got_w.double() - w).abs() <= w_err * w).all()
    L.check(got, *L.reference(x, ids, w, w_err=w_err))
    for _ in range(5):  # on a workspace that was used, the same bits
        again, _, _ = L.run(x, k, ws)
        torch.cuda.synchronize()
        assert torch.equal(again, out)
    # another routing on the same workspace: tokens without an expert, one named twice, a packed y with a residual
    ids2 = ids.flip(0).to(torch.int32).contiguous()
    ids2[0] = -1
    ids2[1] = ids2[1, 0]
    w2 = torch.randn(T, k, generator=L.g, device=cuda_device)
    n = (T + 7) // 8 * 8 * H
    res = torch.zeros((T + 7) // 8 * 8, H, dtype=L.dt, device=cuda_device)
    res[:T] = torch.randn(T, H, generator=L.g, device=cuda_device).to(L.dt)
    y = torch.full((n + 64,), 777.0, dtype=L.dt, device=cuda_device)
    y[:n] = res.reshape(-1, 8, H).transpose(1, 2).reshape(-1)
    out, _, _ = L.run(x, k, ws, ids=ids2, weights=w2, y=y, residual=y, packed=True)
    ref, bound = L.reference(x, ids2.long(), w2)
    r = res[:T].T.double()
    L.check(L.result(out, T, True), ref + r, bound + 2.0 ** -22 * (ref.abs() + r.abs()))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_captured_decode_steps_take_turns_with_one_workspace(cuda_device, int8):
    """Quantiser, int8 projection into strips, expert layer with the strips for residual, quantiser of its strips:
    captured for two layers of different sizes that share a workspace, replayed in turn on new tokens, each step with
    the bits of its own eager run."""
    import torch

    st = torch.cuda.Stream(cuda_device)
    dt, steps = torch.bfloat16, []
    sizes = [(5, 512, 384, 8, 2), (20, 1024, 640, 6, 2)]
    layers = [Layer(cuda_device, H, inter, E, bf16=True, int8=int8, seed=n) for n, (T, H, inter, E, k) in enumerate(sizes)]
    shared = torch.zeros(max(L.workspace(T, k).numel() for L, (T, _, _, _, k) in zip(layers, sizes)), dtype=torch.uint8,
                         device=cuda_device)
    for L, (T, H, inter, E, k) in zip(layers, sizes):
        w, vals, meta, scale = _matrix(L.g, H, H, dt, True, False, cuda_device)
        strips = (T + 7) // 8
        b = dict(x=L.tokens(T), q=torch.empty(T, H, dtype=torch.int8, device=cuda_device), s=torch.empty(T, device=cuda_device),
                 a=torch.zeros(strips * 8 * H, dtype=dt, device=cuda_device), y=torch.zeros(strips * 8 * H, dtype=dt, device=cuda_device),
                 q2=torch.empty(T, H, dtype=torch.int8, device=cuda_device), s2=torch.empty(T, device=cuda_device))

        def step(ws, L=L, T=T, H=H, k=k, b=b, vals=vals, meta=meta, scale=scale):
            s = torch.cuda.current_stream(cuda_device)
            spmm24.quantize_int8(b["x"], T, H, b["q"], b["s"], bf16=True)
            assert spmm24.launch_int8(s, vals, b["q"], meta, b["a"], H, T, H, w_scale=scale, x_scale=b["s"], flags=spmm24.BF16,
                                      alpha=4.0, out_layout=spmm24.OUT_PACKED_B) == 0
            _, ids, w = L.run(b["x"], k, ws, y=b["y"], x_packed=b["a"], residual=b["a"], packed=True, stream=s)
            spmm24.quantize_int8(b["y"], T, H, b["q2"], b["s2"], bf16=True, packed=True)
            return ids, w

        steps.append((step, b, L.workspace(T, k)))
    inputs = [[torch.randn_like(b["x"].float()).to(dt) for _ in range(3)] for _, b, _ in steps]
    want, graphs = [], []
    with torch.cuda.stream(st):
        for (step, b, own), xs in zip(steps, inputs):
            want.append([])
            for x in xs:
                b["x"].copy_(x)
                ids, w = step(own)
                want[-1].append([ids.clone(), w.clone()] + [b[n].clone() for n in ("a", "y", "q2", "s2")])
        st.synchronize()
        for step, b, _ in steps:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                out = step(shared)
            graphs.append((g, out))
        for i in range(3):
            for (step, b, _), (g, out), xs, ref in zip(steps, graphs, inputs, want):
                b["x"].copy_(xs[i])
                for _ in range(4):
                    g.replay()
                for got, r in zip(list(out) + [b[n] for n in ("a", "y", "q2", "s2")], ref[i]):
                    assert torch.equal(got, r)
    torch.cuda.synchronize(cuda_device)
    assert spmm24.device_status(0) == 0
