"""The operators of an int8 2:4 layer and of a mixture-of-experts layer, as timed cases.

Three operators that a decode or prefill step of a 2:4-sparse model calls:

  quantize  16-bit activations -> int8 rows and one scale for each token
  int8      C = act(w_scale[m] x_scale[n] A_sparse B + bias), int8 A (2:4) and B
  moe       a whole mixture-of-experts layer for a few tokens: router, top-k,
            gate / up, act(gate) * up, down, weighted sum; fp16, bf16 or int8
            2:4 experts

`run` computes them in elementary torch operations, or (own) through the
library's entry points.  Weights are made once per layer, in dense form and
in the library's packed form (SpMM_API.h documents both packed formats).
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-repo_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import spmm24

    return spmm24


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decode step, before its q/k/v projections
        {"name": "quantize 1x4096", "op": "quantize", "tokens": 1, "features": 4096, "type": "fp16", "layout": "rows"},
        # a prefill batch of odd length as the previous layer leaves it: strips of eight tokens
        {"name": "quantize 509x4096 strips", "op": "quantize", "tokens": 509, "features": 4096, "type": "fp16",
         "layout": "strips"},
        # a full prefill batch before the down projection
        {"name": "quantize 4096x11008", "op": "quantize", "tokens": 4096, "features": 11008, "type": "bf16",
         "layout": "rows"},
        # decode, one user: weight streaming, the smallest product
        {"name": "int8 4096x1x4096", "op": "int8", "M": 4096, "N": 1, "K": 4096, "type": "fp16", "bias": False,
         "act": "none"},
        # decode, an odd batch, the down projection
        {"name": "int8 4096x13x11008", "op": "int8", "M": 4096, "N": 13, "K": 11008, "type": "bf16", "bias": False,
         "act": "none"},
        # a short ragged prompt, up projection with bias and activation
        {"name": "int8 11008x509x4096 bias silu", "op": "int8", "M": 11008, "N": 509, "K": 4096, "type": "bf16",
         "bias": True, "act": "silu"},
        # prefill
        {"name": "int8 11008x4096x4096", "op": "int8", "M": 11008, "N": 4096, "K": 4096, "type": "fp16", "bias": False,
         "act": "none"},
        # a small layer, odd counts: latency
        {"name": "moe T3 E5k2 1024x640 fp16", "op": "moe", "tokens": 3, "hidden": 1024, "inter": 640, "experts": 5,
         "top_k": 2, "type": "fp16", "int8": False, "norm": True},
        # decode, one user, two large experts of eight
        {"name": "moe T1 E8k2 4096x11008 fp16", "op": "moe", "tokens": 1, "hidden": 4096, "inter": 11008, "experts": 8,
         "top_k": 2, "type": "fp16", "int8": False, "norm": True},
        # decode, a few users, many small experts
        {"name": "moe T8 E64k8 2048x1024 bf16", "op": "moe", "tokens": 8, "hidden": 2048, "inter": 1024, "experts": 64,
         "top_k": 8, "type": "bf16", "int8": False, "norm": False},
        # decode, one user, int8 experts
        {"name": "moe T1 E8k2 4096x11008 int8", "op": "moe", "tokens": 1, "hidden": 4096, "inter": 11008, "experts": 8,
         "top_k": 2, "type": "bf16", "int8": True, "norm": True},
        # the largest batch, every expert in use, int8 experts
        {"name": "moe T32 E8k2 4096x11008 int8", "op": "moe", "tokens": 32, "hidden": 4096, "inter": 11008,
         "experts": 8, "top_k": 2, "type": "fp16", "int8": True, "norm": True},
    ]


def _between(rng, lo, hi, step=1):
    """A multiple of `step`, spread evenly over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step) * step))


def draw(rng):
    op = rng.choice(("quantize", "int8", "int8", "moe", "moe"))
    kind = rng.choice(("fp16", "bf16"))
    if op == "quantize":
        return {"op": op, "tokens": _between(rng, 1, 4096), "features": _between(rng, 128, 11008, 8), "type": kind,
                "layout": rng.choice(("rows", "strips"))}
    if op == "int8":
        act = rng.choice(("none", "relu", "silu", "gelu"))
        return {"op": op, "M": _between(rng, 128, 11008, 16), "N": _between(rng, 1, 4096),
                "K": _between(rng, 256, 4096, 128), "type": kind, "bias": rng.random() < 0.5, "act": act}
    experts = _between(rng, 4, 64)
    int8 = rng.random() < 0.5
    inter = _between(rng, 256, 11008 if experts <= 8 else 1024, 128)
    return {"op": op, "tokens": _between(rng, 1, 32), "hidden": _between(rng, 256, 4096, 128), "inter": inter,
            "experts": experts, "top_k": rng.randint(1, min(8, experts)), "type": kind, "int8": int8,
            "norm": rng.random() < 0.5}


# ----------------------------------------------------------------- inputs
def _prune(w):
    """Magnitude 2:4 along the last axis: (kept values, their places) of each group of four, in order."""
    g = w.reshape(*w.shape[:-1], -1, 4)
    a = g.abs().float()
    ahead = torch.zeros(a.shape, dtype=torch.int8, device=w.device)
    for i in range(4):
        for j in range(4):
            if i != j:
                ahead[..., i] += ((a[..., j] > a[..., i]) | ((a[..., j] == a[..., i]) & (j < i))).to(torch.int8)
    kept = ahead < 2
    first = torch.where(kept[..., 0], 0, torch.where(kept[..., 1], 1, 2))
    last = torch.where(kept[..., 3], 3, torch.where(kept[..., 2], 2, 1))
    place = torch.stack((first, last), -1)
    return g.gather(-1, place), place


def _dense(kept, place):
    """The M x K matrix that the kept values stand for."""
    out = torch.zeros(*kept.shape[:-1], 4, dtype=kept.dtype, device=kept.device)
    return out.scatter_(-1, place, kept).reshape(*kept.shape[:-2], -1)


def _pack16(kept, place):
    """The library's packed form of a 16-bit 2:4 matrix: values and metadata."""
    M, K = kept.shape[0], kept.shape[1] * 4
    vals = kept.reshape(M // 16, 16, K // 16, 8).transpose(1, 2).contiguous().view(torch.int16).reshape(-1)
    shift = torch.arange(0, 16, 2, device=kept.device, dtype=torch.int32)
    word = (place.reshape(M, K // 16, 8).int() << shift).sum(-1, dtype=torch.int32)
    word = word.reshape(M // 16, 2, 8, K // 64, 4).permute(0, 3, 2, 4, 1)  # band, 64-K group, row i, block, half
    word = torch.where(word >= 32768, word - 65536, word).to(torch.int16)
    return vals, word.reshape(-1).contiguous()


def _pack8(kept, place):
    """The library's packed form of an 8-bit 2:4 matrix: values and metadata."""
    M, K = kept.shape[0], kept.shape[1] * 4
    vals = kept.reshape(M // 16, 16, K // 32, 16).transpose(1, 2).contiguous().reshape(-1)
    nibble = (place[..., 0] | place[..., 1] << 2).reshape(M // 16, 16, K // 128, 16, 2)
    byte = (nibble[..., 0] | nibble[..., 1] << 4).to(torch.uint8)
    return vals, byte.transpose(1, 2).contiguous().reshape(-1)


def _strips(x):
    """tokens x features -> the packed B: strips of eight tokens, features x 8 each, pad tokens zero."""
    T, K = x.shape
    p = torch.zeros((T + 7) // 8 * 8, K, dtype=x.dtype, device=x.device)
    p[:T] = x
    return p.reshape(-1, 8, K).transpose(1, 2).contiguous()


def _weights(g, rows, cols, kind, int8):
    """One 2:4 layer: weights N(0, 0.02) pruned by magnitude, dense and packed; int8: with its channel scales."""
    w = torch.empty(rows, cols, device="cuda").normal_(0.0, 0.02, generator=g).to(_TYPES[kind])
    kept, place = _prune(w)
    scale = None
    if int8:
        scale = kept.float().abs().amax((1, 2)) / 127
        kept = (kept.float() / scale[:, None, None]).round().to(torch.int8)
    vals, meta = (_pack8 if int8 else _pack16)(kept, place)
    return {"dense": _dense(kept, place), "values": vals, "meta": meta, "scale": scale}


def _stack(layers):
    """One matrix after another along M: their packed forms follow one another too."""
    return {k: None if layers[0][k] is None else torch.stack([w[k] for w in layers]) if k == "dense" else
            torch.cat([w[k] for w in layers]) for k in layers[0]}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["type"]
    s = {"case": case}
    if case["op"] == "quantize":
        x = torch.empty(case["tokens"], case["features"], device="cuda").normal_(generator=g)
        # activations: a scale of its own for each token, and a few features that stand out
        x *= torch.exp(torch.empty(case["tokens"], 1, device="cuda").normal_(generator=g))
        x[:, ::max(1, case["features"] // 7)] *= 12
        x = x.to(_TYPES[kind])
        s["x"] = x if case["layout"] == "rows" else _strips(x)
        s["q"] = torch.empty(case["tokens"], case["features"], dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(case["tokens"], device="cuda")
    elif case["op"] == "int8":
        M, N, K = case["M"], case["N"], case["K"]
        s["w"] = _weights(g, M, K, kind, True)
        x = torch.empty(N, K, device="cuda").normal_(generator=g)
        s["x_scale"] = x.abs().amax(1) / 127
        s["x"] = (x / s["x_scale"][:, None]).round().to(torch.int8)
        s["bias"] = torch.empty(M, device="cuda").normal_(generator=g).to(_TYPES[kind]) if case["bias"] else None
        s["c"] = torch.empty(M, N, dtype=_TYPES[kind], device="cuda")
    else:
        T, H, inter, E, k = (case[n] for n in ("tokens", "hidden", "inter", "experts", "top_k"))
        # RMS-normed tokens
        s["x"] = torch.empty(T, H, device="cuda").normal_(generator=g).to(_TYPES[kind])
        s["x_packed"] = _strips(s["x"])
        s["router"] = torch.empty(E, H, device="cuda").normal_(0.0, 0.02, generator=g).to(_TYPES[kind])
        s["gate_up"] = _stack([_weights(g, 2 * inter, H, kind, case["int8"]) for _ in range(E)])
        s["down"] = _stack([_weights(g, H, inter, kind, case["int8"]) for _ in range(E)])
        s["y"] = torch.empty(H, T, dtype=_TYPES[kind], device="cuda")
        s["ids"] = torch.empty(T, k, dtype=torch.int32, device="cuda")
        s["weights"] = torch.empty(T, k, device="cuda")
        # int8: at most 4 bytes and a byte for each value between the two products, and the partial sums
        s["workspace"] = torch.zeros(_workspace(case), dtype=torch.uint8, device="cuda")
    return s


def _workspace(case):
    """Bytes of a workspace that holds every layer of these sizes (a program asks the library for the exact number)."""
    slots = min(case["experts"], case["tokens"] * case["top_k"])
    return (32 << 20) + slots * 32 * (case["inter"] + 128) * 5 + 4096 * case["experts"]


# -------------------------------------------------------------- one pass
def run(s):
    return {"quantize": _quantize, "int8": _int8, "moe": _moe}[s["case"]["op"]](s)


def _act(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _rows_to_int8(x):
    """Rows of x -> int8 values (as floats) and scales; 64 bits decide the values next to a border."""
    top = x.abs().amax(-1, keepdim=True).double()
    q = torch.where(top > 0, x.double() * 127 / top, torch.zeros_like(top)).round()
    return q, (top / 127).float()


def _quantize(s):
    case = s["case"]
    T, K = case["tokens"], case["features"]
    if own:
        lib = _library()
        lib.quantize_int8(s["x"], T, K, s["q"], s["scale"], bf16=case["type"] == "bf16", packed=case["layout"] == "strips")
        return {"q": s["q"], "scale": s["scale"]}
    x = s["x"] if case["layout"] == "rows" else s["x"].transpose(1, 2).reshape(-1, K)[:T]
    q, scale = _rows_to_int8(x)
    return {"q": q.to(torch.int8), "scale": scale[:, 0]}


def _int8(s):
    case, w = s["case"], s["w"]
    M, N, K = case["M"], case["N"], case["K"]
    if own:
        lib = _library()
        acts = {"none": lib.ACT_NONE, "relu": lib.ACT_RELU, "silu": lib.ACT_SILU, "gelu": lib.ACT_GELU}
        rc = lib.launch_int8(torch.cuda.current_stream(), w["values"], s["x"], w["meta"], s["c"], M, N, K,
                             w_scale=w["scale"], x_scale=s["x_scale"],
                             flags=lib.STATIC_WEIGHTS | (lib.BF16 if case["type"] == "bf16" else 0), bias=s["bias"],
                             activation=acts[case["act"]])
        if rc:
            raise lib.SpmmError(rc, "spmm24_launch_int8")
        return s["c"]
    y = (w["dense"].float() @ s["x"].float().T) * w["scale"][:, None] * s["x_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()[:, None]
    return _act(y, case["act"]).to(_TYPES[case["type"]])


def _moe(s):
    case = s["case"]
    T, H, inter, E, k = (case[n] for n in ("tokens", "hidden", "inter", "experts", "top_k"))
    if own:
        lib = _library()
        flags = (lib.BF16 if case["type"] == "bf16" else 0) | (lib.MOE_INT8 if case["int8"] else 0)
        rc = lib.launch_moe(torch.cuda.current_stream(), s["x_packed"], s["router"], s["gate_up"]["values"],
                            s["gate_up"]["meta"], s["down"]["values"], s["down"]["meta"], s["y"], T, H, inter, E, k,
                            s["workspace"], flags=flags, gate_up_scale=s["gate_up"]["scale"],
                            down_scale=s["down"]["scale"], topk_ids=s["ids"], topk_weights=s["weights"],
                            norm_topk=case["norm"])
        if rc:
            raise lib.SpmmError(rc, "spmm24_launch_moe")
        return {"y": s["y"], "ids": s["ids"], "weights": s["weights"]}
    x = s["x"].float()
    logits = x @ s["router"].float().T
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k]
    e = torch.exp(logits - logits.amax(1, keepdim=True))
    weights = (e / e.sum(1, keepdim=True)).gather(1, ids)
    if case["norm"]:
        weights = weights / weights.sum(1, keepdim=True)
    x_scale = torch.ones(T, 1, device=x.device)
    if case["int8"]:
        q, x_scale = _rows_to_int8(s["x"])
        x = q.float()
    # few pairs of a token and an expert: those alone; else every expert on every token
    pairs = T * k < E
    gate_up, down = s["gate_up"], s["down"]
    pick = ids.reshape(-1) if pairs else slice(None)
    cols = x.repeat_interleave(k, 0)[:, :, None] if pairs else x.T
    col_scale = x_scale.repeat_interleave(k, 0)[:, :, None] if pairs else x_scale.T
    gu = gate_up["dense"][pick].float() @ cols
    if case["int8"]:
        gu = gu * gate_up["scale"].reshape(E, 2 * inter, 1)[pick] * col_scale
    h = _act(gu[:, :inter], "silu") * gu[:, inter:]
    if case["int8"]:
        top = h.abs().amax(1, keepdim=True)
        h = torch.where(top > 0, h * 127 / top, torch.zeros_like(top)).round()
        y = (down["dense"][pick].float() @ h) * down["scale"].reshape(E, H, 1)[pick] * (top / 127)
    else:
        h = h.to(_TYPES[case["type"]]).float()  # a 16-bit product takes 16-bit operands
        y = down["dense"][pick].float() @ h
    if pairs:
        y = (y.reshape(T, k, H) * weights[:, :, None]).sum(1).T
    else:
        each = torch.zeros(T, E, device=x.device).scatter_(1, ids, weights)
        y = (y * each.T[:, None, :]).sum(0)
    return {"y": y.to(_TYPES[case["type"]]), "ids": ids.int(), "weights": weights}


# ------------------------------------------------------------- definition
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        T, K = case["tokens"], case["features"]
        x = (s["x"] if case["layout"] == "rows" else s["x"].permute(0, 2, 1).reshape(-1, K)[:T]).double()
        top = x.abs().max(1).values
        return {"q": None, "scale": top / 127}
    if case["op"] == "int8":
        w = s["w"]["dense"].double() * s["w"]["scale"].double()[:, None]
        y = torch.einsum("mk,nk->mn", w, s["x"].double() * s["x_scale"].double()[:, None])
        if s["bias"] is not None:
            y += s["bias"].double()[:, None]
        return _act(y, case["act"])
    H, inter, E, k = (case[n] for n in ("hidden", "inter", "experts", "top_k"))
    x = s["x"].double()
    p = torch.softmax(torch.einsum("th,eh->te", x, s["router"].double()), 1)
    weights, ids = p.topk(k, 1)
    if case["norm"]:
        weights = weights / weights.sum(1, keepdim=True)
    if case["int8"]:  # the activations that the products are defined on
        x = (x / (x.abs().amax(1, keepdim=True) / 127)).round() * (x.abs().amax(1, keepdim=True) / 127)
    y = torch.zeros(H, case["tokens"], dtype=torch.double, device="cuda")
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        gu, down = s["gate_up"]["dense"][e].double(), s["down"]["dense"][e].double()
        if case["int8"]:
            gu *= s["gate_up"]["scale"].reshape(E, 2 * inter)[e].double()[:, None]
            down *= s["down"]["scale"].reshape(E, H)[e].double()[:, None]
        g, u = (gu @ x[t].T).split(inter)
        h = g * torch.sigmoid(g) * u
        if case["int8"]:
            step = h.abs().amax(0) / 127
            h = (h / step).round() * step
        y[:, t] += (down @ h) * weights[t, j]
    return {"y": y, "ids": None, "weights": weights}


def work(case):
    if case["op"] == "quantize":
        n = case["tokens"] * case["features"]
        return {"bytes": 3 * n + 4 * case["tokens"], "flops": 3 * n}
    if case["op"] == "int8":
        M, N, K = case["M"], case["N"], case["K"]
        # values and metadata of the kept half of A, B, scales, C; the kept products alone
        return {"bytes": M * K * 5 / 8 + N * K + 4 * (M + N) + 2 * M * N, "flops": M * N * K}
    T, H, inter, E, k = (case[n] for n in ("tokens", "hidden", "inter", "experts", "top_k"))
    used = E * (1 - (1 - k / E) ** T)  # experts that T tokens meet
    weight = 5 / 8 if case["int8"] else 9 / 8
    return {"bytes": used * 3 * inter * H * weight + 2 * E * H + 4 * T * H, "flops": T * k * 3 * inter * H + 2 * T * E * H}
