"""spmm24_launch_moe against the layer's formulas in 64 bits (torch doubles on
the same device, dense weights, one expert after another)."""
import numpy as np
import pytest

import spmm24
from int8_problems import act64

pytestmark = pytest.mark.gpu


def _act(y, act):
    import torch

    return torch.from_numpy(act64(y.cpu().numpy(), act)).to(y.device)


def _slope(act):
    return 1.13 if act >= 2 else 1.0


def _strips(x):
    import torch

    T, H = x.shape
    p = torch.full(((T + 7) // 8 * 8, H), float("nan"), dtype=x.dtype, device=x.device)  # pad tokens are not used
    p[:T] = x
    return p.reshape(-1, 8, H).transpose(1, 2).contiguous()


def _matrix(g, rows, cols, dt, int8, integers, device):
    """A random 2:4 matrix: (dense doubles, values, metadata, scales)."""
    import torch

    bf16 = dt == torch.bfloat16
    if integers:
        w = torch.randint(-1, 2, (rows, cols), generator=g, device=device).to(dt)
    else:
        w = (torch.randn(rows, cols, generator=g, device=device) * 0.02).to(dt)
    spmm24.prune_2of4_device(w, rows, cols, bf16=bf16)
    if not int8:
        vals, meta, bad = spmm24.pack_a_device(w, rows, cols)
        assert bad == 0
        return w.double(), vals, meta, None
    q, scale = spmm24.quantize_int8(w, rows, cols, bf16=bf16)
    vals, meta = spmm24.pack_a_int8_device(q, rows, cols)
    return q.double() * scale.double()[:, None], vals, meta, scale


class Layer:
    def __init__(self, device, H, inter, E, bf16=False, int8=False, integers=False, seed=0):
        import torch

        self.device, self.H, self.inter, self.E, self.bf16, self.int8 = device, H, inter, E, bf16, int8
        self.dt = torch.bfloat16 if bf16 else torch.float16
        self.g = torch.Generator(device=device).manual_seed(seed)
        self.gu = _matrix(self.g, E * 2 * inter, H, self.dt, int8, integers, device)
        self.dn = _matrix(self.g, E * H, inter, self.dt, int8, integers, device)
        self.router = (torch.randn(E, H, generator=self.g, device=device) * 0.05).to(self.dt)
        self.flags = (spmm24.BF16 if bf16 else 0) | (spmm24.MOE_INT8 if int8 else 0)

    def tokens(self, T, integers=False):
        import torch

        if integers:
            return torch.randint(-1, 2, (T, self.H), generator=self.g, device=self.device).to(self.dt)
        return torch.randn(T, self.H, generator=self.g, device=self.device).to(self.dt)

    def workspace(self, T, k):
        import torch

        return torch.zeros(spmm24.moe_workspace_bytes(T, self.H, self.inter, self.E, k, self.flags), dtype=torch.uint8,
                           device=self.device)

    def run(self, x, k, ws, *, ids=None, weights=None, stream=None, y=None, packed=False, x_packed=None, **kw):
        """(y, ids, weights) of one launch; ids and weights given: no router."""
        import torch

        T = x.shape[0]
        given = ids is not None
        if ids is None:
            ids = torch.full((T, k), -7, dtype=torch.int32, device=self.device)
            weights = torch.full((T, k), -7.0, device=self.device)
        n = (T + 7) // 8 * 8 * self.H if packed else T * self.H
        if y is None:
            y = torch.full((n + 64,), 777.0, dtype=self.dt, device=self.device)
        xp = _strips(x) if x_packed is None else x_packed
        stream = stream or torch.cuda.current_stream(self.device)
        rc = spmm24.launch_moe(stream, xp, None if given else self.router, self.gu[1], self.gu[2], self.dn[1], self.dn[2],
                               y, T, self.H, self.inter, self.E, k, ws, flags=self.flags, gate_up_scale=self.gu[3],
                               down_scale=self.dn[3], topk_ids=ids, topk_weights=weights,
                               out_layout=spmm24.OUT_PACKED_B if packed else spmm24.OUT_ROW_MAJOR, **kw)
        assert rc == 0, spmm24._lib.spmm24_last_error().decode()
        return y, ids, weights

    def result(self, out, T, packed=False):
        """The H x T doubles of a launch's y; checks what lies behind it."""
        import torch

        torch.cuda.synchronize(self.device)
        assert spmm24.device_status(self.device.index or 0) == 0
        n = out.numel() - 64
        assert (out[n:] == 777.0).all(), "wrote behind y"
        if packed:
            full = out[:n].reshape(-1, self.H, 8).permute(1, 0, 2).reshape(self.H, -1)
            assert not full[:, T:].any(), "pad columns of a packed y must be zero"
            return full[:, :T].double()
        return out[:n].reshape(self.H, T).double()

    def routed(self, x, k, norm):
        """(ids, weights, bound of the weights' relative error) by the formula."""
        import torch

        logits = x.double() @ self.router.double().T
        s = x.double().abs() @ self.router.double().abs().T
        # fp32 sums of H products in at most H / 256 * 8 + 5 + 32 steps of 2^-24 relative to the terms' sizes
        err = ((self.H / 32 + 40) * 2.0 ** -24 * s).max().item()
        order = torch.sort(logits, dim=1, descending=True, stable=True)
        ids = order.indices[:, :k]
        if k < self.E:  # the seeds leave no choice within the sums' error
            assert (order.values[:, k - 1] - order.values[:, k]).min() > 2 * err
        if k > 1:
            assert (order.values[:, : k - 1] - order.values[:, 1:k]).min() > 2 * err
        p = torch.softmax(logits, 1).gather(1, ids)
        if norm:
            p = p / p.sum(1, keepdim=True)
        # exp(l - max) of a sum off by err each; exp, sum (256 terms) and division to 2^-20
        return ids, p, 4 * err + 2.0 ** -19

    def reference(self, x, ids, weights, act=2, w_err=0.0):
        """(y, bound) before the epilogue, fp64: H x T each."""
        import torch

        T, k = ids.shape
        H, I, E = self.H, self.inter, self.E
        gu, dn = self.gu[0].reshape(E, 2 * I, H), self.dn[0].reshape(E, H, I)
        x = x.double()
        if self.int8:
            top = x.abs().amax(1, keepdim=True)
            sx = (top / 127).float().double()
            x = torch.where(top > 0, (127 * x / top).round(), torch.zeros_like(top)) * sx
        y = torch.zeros(H, T, dtype=torch.double, device=self.device)
        bound = torch.zeros_like(y)
        half = 2.0 ** (-8 if self.bf16 else -11)
        tiny = 0.0 if self.bf16 else 2.0 ** -25
        c = 2.0 ** -14  # fp32 sums of the tensor core, relative to the terms' sizes: fewer than 2^9 steps of 2^-23
        for e in range(E):
            t, j = (ids == e).nonzero(as_tuple=True)
            if not len(t):
                continue
            w = weights[t, j].double()
            z = gu[e] @ x[t].T
            gate, up = z[:I], z[I:]
            if self.int8:
                dz = 4 * 2.0 ** -24 * z.abs()  # exact sums; conversion, two scales
            else:
                dz = c * (gu[e].abs() @ x[t].abs().T)
            a = _act(gate, act)
            h = a * up
            dh = _slope(act) * dz[:I] * (up.abs() + dz[I:]) + a.abs() * dz[I:] + 2.0 ** -20 * h.abs()
            if self.int8:
                top = h.abs().amax(0, keepdim=True)
                dtop = dh.amax(0, keepdim=True)
                s = top / 127
                v = torch.where(top > 0, 127 * h / top, torch.zeros_like(top))
                q = v.round()
                dv = torch.where(top > 0, 127 * dh / top + v.abs() * (dtop / top + 2.0 ** -22), torch.zeros_like(top))
                flips = (((v - v.floor()) - 0.5).abs() <= dv).double()  # next to a tie: one step either way
                ds = s * (dtop / top.clamp(min=1e-300) + 2.0 ** -22)
                d = dn[e] @ (q * s)
                dd = dn[e].abs() @ (flips * s + q.abs() * ds) + 4 * 2.0 ** -24 * d.abs()
            else:
                hr = h.to(self.dt).double()
                dh = dh * (1 + 2 * half) + 2 * half * h.abs() + tiny  # may round to the next value
                d = dn[e] @ hr
                dd = dn[e].abs() @ dh + c * (dn[e].abs() @ (hr.abs() + dh))
            y.index_add_(1, t, w * d)
            bound.index_add_(1, t, w.abs() * (dd + (w_err + 2.0 ** -21) * (d.abs() + dd)))
        return y, bound

    def check(self, got, y, bound):
        half = 2.0 ** (-8 if self.bf16 else -11)
        tol = bound * (1 + half) + half * y.abs() + (0 if self.bf16 else 2.0 ** -25)
        bad = ~((got - y).abs() <= tol)
        assert not bad.any(), (int(bad.sum()), float((got - y).abs().max()), float(tol.max()))
        # the bound sums every error with its worst sign; a misplaced column or
        # expert is off by the size of y itself
        assert (got - y).norm() <= 0.05 * y.norm() + 1e-12


SHAPES = [(1, 128, 128, 1, 1), (3, 1024, 640, 5, 2), (8, 256, 384, 64, 8), (9, 128, 256, 7, 3), (16, 384, 896, 4, 4),
          (17, 384, 640, 6, 2), (32, 512, 1408, 16, 4), (32, 256, 256, 256, 16), (2, 4096, 2048, 8, 2),
          (24, 2176, 128, 33, 5), (2, 24576, 128, 3, 2), (1, 128, 8192, 5, 3), (11, 4096, 1408, 12, 3)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "T%d-%dx%d-E%dk%d" % s)
@pytest.mark.parametrize("kind", ["fp16", "bf16", "int8-fp16", "int8-bf16"])
def test_layer_matches_the_formula(cuda_device, shape, kind):
    import torch

    T, H, inter, E, k = shape
    for norm in (True, False):
        L = Layer(cuda_device, H, inter, E, bf16=kind.endswith("bf16"), int8=kind.startswith("int8"), seed=T + E)
        x = L.tokens(T)
        ids, w, w_err = L.routed(x, k, norm)
        ws = L.workspace(T, k)
        out, got_ids, got_w = L.run(x, k, ws, norm_topk=norm)
        got = L.result(out, T)
        assert torch.equal(got_ids.long(), ids)
        assert ((got_w.double() - w).abs() <= w_err * w).all()
        L.check(got, *L.reference(x, ids, w, w_err=w_err))
        # the same call again, on a workspace that was used: the same bits
        again, ids2, w2 = L.run(x, k, ws, norm_topk=norm)
        torch.cuda.synchronize()
        assert torch.equal(again, out) and torch.equal(ids2, got_ids) and torch.equal(w2, got_w)


@pytest.mark.parametrize("shape", [(5, 192, 320, 9, 2), (12, 64, 64, 3, 3), (32, 448, 1088, 12, 2)],
                         ids=lambda s: "T%d-%dx%d-E%dk%d" % s)
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
def test_half_filled_last_stages(cuda_device, shape, bf16):
    """An odd number of 64-K groups in hidden or inter (16-bit experts only)."""
    T, H, inter, E, k = shape
    L = Layer(cuda_device, H, inter, E, bf16=bf16, seed=T)
    x = L.tokens(T)
    ids, w, w_err = L.routed(x, k, True)
    out, _, _ = L.run(x, k, L.workspace(T, k))
    L.check(L.result(out, T), *L.reference(x, ids, w, w_err=w_err))


@pytest.mark.parametrize("T,H,inter,E", [(1, 256, 256, 4), (7, 512, 320, 3), (32, 1024, 640, 20)])
def test_integers_are_exact(cuda_device, T, H, inter, E):
    """Weights and tokens of -1, 0, 1, ReLU, one expert each: every sum is an
    integer below 2^24, so only the two roundings to fp16 that the layer defines
    (h, above 2048, and y) take part, and the result is exact."""
    import torch

    L = Layer(cuda_device, H, inter, E, integers=True, seed=T)
    x = L.tokens(T, integers=True)
    ids = torch.randint(0, E, (T, 1), generator=L.g, device=cuda_device, dtype=torch.int32)
    w = torch.full((T, 1), 2.0 ** -4, device=cuda_device)
    out, _, _ = L.run(x, 1, L.workspace(T, 1), ids=ids, weights=w, activation=spmm24.ACT_RELU)
    got = L.result(out, T)
    z = torch.einsum("trh,th->tr", L.gu[0].reshape(E, 2 * inter, H)[ids[:, 0].long()], x.double())
    h = z[:, :inter].clamp(min=0) * z[:, inter:]
    h = h.to(torch.float16).double()
    y = torch.einsum("thi,ti->ht", L.dn[0].reshape(E, H, inter)[ids[:, 0].long()], h) / 16
    assert torch.equal(got, y.to(torch.float16).double())


@pytest.mark.parametrize("int8", [False, True], ids=["fp16", "int8"])
@pytest.mark.parametrize("act", [0, 1, 2, 3], ids=["none", "relu", "silu", "gelu"])
def test_activations_epilogues_and_layouts(cuda_device, act, int8):
    import torch

    for T, packed in ((8, False), (13, False), (13, True), (24, True)):
        L = Layer(cuda_device, 256, 384, 6, int8=int8, seed=act)
        x = L.tokens(T)
        ids, w, w_err = L.routed(x, 2, True)
        res = torch.randn(256, T, generator=L.g, device=cuda_device).half()
        bias = torch.randn(256, generator=L.g, device=cuda_device).half()
        pad = torch.zeros(256, (T + 7) // 8 * 8, dtype=torch.float16, device=cuda_device)
        pad[:, :T] = res
        layout = pad.reshape(256, -1, 8).transpose(0, 1).reshape(-1) if packed else res.reshape(-1)
        y = torch.full((layout.numel() + 64,), 777.0, dtype=torch.float16, device=cuda_device)
        y[: layout.numel()] = layout  # the residual is y itself
        out, _, _ = L.run(x, 2, L.workspace(T, 2), y=y, residual=y, bias=bias, alpha=0.5, packed=packed, activation=act)
        ref, bound = L.reference(x, ids, w, act=act, w_err=w_err)
        ref = 0.5 * ref + bias.double()[:, None] + res.double()
        size = ref.abs() + bias.double().abs()[:, None] + res.double().abs()
        L.check(L.result(out, T, packed), ref, 0.5 * bound + 2.0 ** -22 * size)


@pytest.mark.parametrize("int8", [False, True], ids=["fp16", "int8"])
def test_given_experts(cuda_device, int8):
    """Padded tokens (no expert), ids out of range, the same expert twice,
    weights of zero and of either sign; then no token with an expert at all."""
    import torch

    T, E, k = 11, 9, 3
    L = Layer(cuda_device, 256, 384, E, int8=int8, seed=5)
    x = L.tokens(T)
    ids = torch.randint(0, E, (T, k), generator=L.g, device=cuda_device, dtype=torch.int32)
    ids[0] = -1
    ids[1] = torch.tensor([4, 4, 2])
    ids[2] = torch.tensor([E, 3, -5])
    ids[3] = torch.tensor([2 ** 31 - 1, -2 ** 31, 8])
    ids[10] = torch.tensor([-1, -1, 0])
    w = torch.randn(T, k, generator=L.g, device=cuda_device)
    w[4, 0] = 0.0
    ws = L.workspace(T, k)
    before = (ids.clone(), w.clone())
    out, _, _ = L.run(x, k, ws, ids=ids, weights=w)
    got = L.result(out, T)
    assert torch.equal(ids, before[0]) and torch.equal(w, before[1])
    y, bound = L.reference(x, ids.long(), w)
    L.check(got, y, bound)
    assert not got[:, 0].any()
    ids.fill_(-1)
    res = torch.randn(256 * T, device=cuda_device).half()
    out, _, _ = L.run(x, k, ws, ids=ids, weights=w, residual=res)
    assert torch.equal(L.result(out, T), res.reshape(256, T).double())
    # and the workspace still serves
    out, _, _ = L.run(x, k, ws, ids=before[0], weights=w)
    assert torch.equal(L.result(out, T), got)


def test_ties_go_to_the_lower_expert(cuda_device):
    import torch

    E, k, T = 70, 4, 5
    L = Layer(cuda_device, 128, 128, E, seed=1)
    L.router[:] = L.router[0]  # every expert the same logit
    _, ids, w = L.run(L.tokens(T), k, L.workspace(T, k))
    assert torch.equal(ids.cpu(), torch.arange(k, dtype=torch.int32).expand(T, k))
    assert torch.allclose(w, torch.full_like(w, 0.25), rtol=1e-6, atol=0)
    L.router[40:] = 0  # two levels: +-0 and the rest
    L.router[:40] = 0
    L.router[10, 0], L.router[69, 0] = 1, 1
    x = torch.zeros(T, 128, dtype=torch.float16, device=cuda_device)
    x[:, 0] = 1
    x[1, 0] = -1
    _, ids, _ = L.run(x, k, L.workspace(T, k))
    assert ids[0].tolist() == [10, 69, 0, 1] and ids[1].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("int8", [False, True], ids=["fp16", "int8"])
def test_infinities_and_nan_stay_in_their_token(cuda_device, int8):
    import torch

    T, k = 10, 2
    L = Layer(cuda_device, 256, 256, 8, int8=int8, seed=2)
    x = L.tokens(T)
    ids, w, w_err = L.routed(x, k, True)
    y, bound = L.reference(x, ids, w, w_err=w_err)
    x[3, 17] = float("inf")
    x[9, 0] = float("nan")
    out, got_ids, got_w = L.run(x, k, L.workspace(T, k))
    got = L.result(out, T)
    keep = [t for t in range(T) if t not in (3, 9)]
    L.check(got[:, keep], y[:, keep], bound[:, keep])
    assert torch.isnan(got[:, 9]).all() and torch.isnan(got_w[9]).all()
    assert not torch.isfinite(got[:, 3]).any()
    assert torch.equal(got_ids[keep].long(), ids[keep])


def test_large_logits_and_zero_tokens(cuda_device):
    import torch

    L = Layer(cuda_device, 128, 128, 6, int8=True, seed=8)
    L.router *= 400  # logits of hundreds: all weight on the first expert
    x = L.tokens(4)
    x[2] = 0  # a padded token of zeros
    out, ids, w = L.run(x, 3, L.workspace(4, 3), norm_topk=False)
    got = L.result(out, 4)
    assert torch.isfinite(got).all() and not got[:, 2].any()
    assert ids[2].tolist() == [0, 1, 2] and torch.allclose(w[2], torch.full((3,), 1 / 6, device=cuda_device), rtol=1e-6)
    assert (w[[0, 1, 3], 0] > 0.99).all()


def test_layers_of_other_sizes_share_a_workspace(cuda_device):
    """One zeroed workspace, launches of different sizes and types in turn, each
    as on a workspace of its own."""
    import torch

    cases = [(3, 1024, 640, 5, 2, False), (32, 256, 256, 64, 8, True), (1, 512, 1408, 4, 1, False),
             (17, 384, 640, 6, 2, True), (3, 1024, 640, 5, 2, False)]
    layers = [(Layer(cuda_device, H, i, E, int8=q, seed=n), T, k) for n, (T, H, i, E, k, q) in enumerate(cases)]
    xs = [L.tokens(T) for L, T, _ in layers]
    own = [L.run(x, k, L.workspace(T, k))[0] for (L, T, k), x in zip(layers, xs)]
    shared = torch.zeros(max(L.workspace(T, k).numel() for L, T, k in layers), dtype=torch.uint8, device=cuda_device)
    for _ in range(3):
        got = [L.run(x, k, shared)[0] for (L, T, k), x in zip(layers, xs)]
    torch.cuda.synchronize()
    for a, b in zip(got, own):
        assert torch.equal(a, b)


def test_other_stream_and_graph(cuda_device):
    """Captured once, replayed on new tokens with other routings; two captured
    graphs with a workspace each on two streams at once."""
    import torch

    T, k = 6, 2
    L = Layer(cuda_device, 1024, 640, 8, bf16=True, seed=3)
    xs = [L.tokens(T) for _ in range(4)]
    want = [L.run(x, k, L.workspace(T, k)) for x in xs]
    torch.cuda.synchronize()
    runs = []
    for n in range(2):
        s = torch.cuda.Stream(cuda_device)
        ws, xp = L.workspace(T, k), _strips(xs[0])
        y = torch.zeros(T * 1024 + 64, dtype=L.dt, device=cuda_device)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            _, ids, w = L.run(xs[0], k, ws, y=y, x_packed=xp, stream=s)
        runs.append((graph, s, xp, y, ids, ws))  # a graph's workspace lives as long as the graph
    torch.cuda.synchronize()
    for i, x in enumerate(xs):
        for graph, s, xp, y, ids, _ in runs:
            with torch.cuda.stream(s):
                xp.copy_(_strips(x))
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, s, xp, y, ids, _ in runs:
            assert torch.equal(y[:-64], want[i][0][:-64]) and torch.equal(ids, want[i][1])
    assert spmm24.device_status(0) == 0


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_decode_step(cuda_device, int8):
    """As used together: an int8 projection whose output strips are the expert
    layer's tokens, the layer with the residual, its strips quantised for the
    next int8 projection."""
    import torch

    T, H, k = 5, 512, 2
    L = Layer(cuda_device, H, 384, 8, bf16=True, int8=int8, seed=4)
    dt = torch.bfloat16
    P = _matrix(L.g, H, H, dt, True, False, cuda_device)
    x = L.tokens(T)
    st = torch.cuda.current_stream(cuda_device)
    q, s = spmm24.quantize_int8(x, T, H, bf16=True)
    a = torch.zeros(1, H, 8, dtype=dt, device=cuda_device)
    rc = spmm24.launch_int8(st, P[1], q, P[2], a, H, T, H, w_scale=P[3], x_scale=s, flags=spmm24.BF16, alpha=4.0,
                            out_layout=spmm24.OUT_PACKED_B)
    assert rc == 0
    ws = L.workspace(T, k)
    y = torch.full((8 * H + 64,), 777.0, dtype=dt, device=cuda_device)
    tok = a[0, :, :T].T.contiguous()
    _, ids, w = L.run(tok, k, ws, y=y, x_packed=a, residual=a, packed=True)
    q2, s2 = spmm24.quantize_int8(y, T, H, bf16=True, packed=True)
    torch.cuda.synchronize()
    ref_a = 4 * (P[0] @ (q.double() * s.double()[:, None]).T)
    assert ((tok.double().T - ref_a).abs() <= 2.0 ** -7.9 * ref_a.abs()).all()
    rids, rw, w_err = L.routed(tok, k, True)
    assert torch.equal(ids.long(), rids)
    ref, bound = L.reference(tok, rids, rw, w_err=w_err)
    ref = ref + tok.double().T
    got = L.result(y, T, packed=True)
    L.check(got, ref, bound + 2.0 ** -23 * (ref.abs() + tok.double().T.abs()))
    top = got.abs().amax(0)
    assert torch.equal(q2.double(), (127 * got / top).round().T) and torch.equal(s2, (top / 127).float())
