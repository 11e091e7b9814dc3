"""Performance cases of the experts' matrix products over ragged groups of rows (bf16, with
gradients) and of products with 4-bit weights (codes with group scales, or MXFP4): quantizer,
dense product and product grouped by expert.

With `own` the passes go through the library (`hkq`); without it they are elementary torch
operations in float32. `prepare` keeps what a program keeps between steps: weights, routing of
the batch, output buffers, workspaces. `exact` repeats the definitions in float64.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16

# (hidden, ffn, experts, experts per token) of the mixture layers that the benchmark and the tests use
MIXTURES = [(4096, 14336, 8, 2), (2048, 1408, 64, 6)]
# (hidden, ffn) of the dense layers
LAYERS = [(4096, 14336), (2048, 2816), (2048, 1408)]
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # down projections of 24 sequences that decode, two experts each: the weights' way from memory
        {"name": "grouped_decode", "kind": "grouped", "M": 48, "E": 8, "active": 8, "N": 4096, "K": 14336},
        # gate and up projections of a small layer's many experts over an odd prefill chunk
        {"name": "grouped_chunk", "kind": "grouped", "M": 6006, "E": 64, "active": 64, "N": 2816, "K": 2048},
        # the training forward of a large layer's gate and up projections
        {"name": "grouped_train", "kind": "grouped", "M": 8192, "E": 8, "active": 8, "N": 28672, "K": 4096},
        # backward of a small layer's down projections, an odd number of tokens, some experts without any
        {"name": "grouped_bwd_small", "kind": "grouped_bwd", "M": 1806, "E": 64, "active": 59, "N": 2048, "K": 1408},
        # backward of a large layer's gate and up projections, a whole micro-batch
        {"name": "grouped_bwd_train", "kind": "grouped_bwd", "M": 8192, "E": 8, "active": 8, "N": 28672, "K": 4096},
        # quantizing a small projection in groups of 32, and a large one with zero points, as a model is loaded
        {"name": "w4_quant_small", "kind": "w4_quant", "N": 1408, "K": 2048, "group": 32, "zeros": False},
        {"name": "w4_quant_large", "kind": "w4_quant", "N": 14336, "K": 4096, "group": 128, "zeros": True},
        # one token through an attention projection: latency
        {"name": "w4_token", "kind": "w4", "M": 1, "N": 4096, "K": 4096, "group": 128, "zeros": False},
        # decode of 16 sequences through gate and up projections with zero points
        {"name": "w4_decode", "kind": "w4", "M": 16, "N": 28672, "K": 4096, "group": 128, "zeros": True},
        # a prefill of two thousand tokens through the same layer's down projection
        {"name": "w4_prefill", "kind": "w4", "M": 2048, "N": 4096, "K": 14336, "group": 128, "zeros": False},
        # one token through its two experts of eight, MXFP4 weights
        {"name": "w4_grouped_token", "kind": "w4_grouped", "M": 2, "E": 8, "active": 2, "topk": 2, "N": 28672, "K": 4096,
         "group": 0, "zeros": False},
        # an odd prefill chunk through many small experts
        {"name": "w4_grouped_chunk", "kind": "w4_grouped", "M": 6006, "E": 64, "active": 64, "topk": 6, "N": 2816, "K": 2048,
         "group": 64, "zeros": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["grouped", "grouped", "grouped_bwd", "w4_quant", "w4", "w4", "w4_grouped", "w4_grouped"])
    c = {"kind": kind}
    if kind in ("w4_quant", "w4"):
        group = rng.choice([32, 64, 128] if kind == "w4_quant" else [0, 32, 64, 128, 128])
        if rng.random() < 0.5:
            N, K = rng.choice(LAYERS)
            N, K = (N, K) if rng.random() < 0.5 else (K, N)
        else:
            N, K = 4 * _log_int(rng, 32, 3584), (group or 32) * _log_int(rng, 4, 8192 // (group or 32))
        zeros = group > 0 and rng.random() < 0.5
        if kind == "w4":
            c["M"] = _log_int(rng, 1, 2048)
        return {**c, "N": N, "K": K, "group": group, "zeros": zeros}
    if rng.random() < 0.5:
        D, F, E, topk = rng.choice(MIXTURES)
        N, K = (2 * F, D) if rng.random() < 0.5 else (D, F)
    else:  # generic sizes; fewer experts of the larger ones
        E, topk = 2 ** rng.randint(1, 6), rng.randint(1, 4)
        N, K = 8 * _log_int(rng, 16, 1024), 8 * _log_int(rng, 16, 512)
    tokens = _log_int(rng, 1, 8192 // topk)
    M = tokens * topk
    active = min(E, M) if rng.random() < 0.5 else rng.randint((min(E, M) + 1) // 2, min(E, M))
    c.update(M=M, E=E, active=active, N=N, K=K)
    if kind == "w4_grouped":
        c["group"] = rng.choice([0, 32, 64, 128])
        c["zeros"] = c["group"] > 0 and rng.random() < 0.5
        c["topk"] = topk
        unit = c["group"] or 32
        c["K"] = (K + unit - 1) // unit * unit
    return c


# ---------------------------------------------------------------------------
# inputs (from the seed alone)
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1000 * (int(seed) % (1 << 40)))


def _randn(shape, g, std=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).mul_(std).to(BF16)


def _counts(c, seed):
    """Rows of each expert: `active` experts, some more popular than others, share M rows; the others have none."""
    rng = random.Random(int(seed) * 7919 + 13)
    who = sorted(rng.sample(range(c["E"]), c["active"]))
    share = [math.exp(0.7 * rng.gauss(0.0, 1.0)) for _ in who]
    free, total = c["M"] - c["active"], sum(share)
    edge, seen = [0], 0.0
    for s in share:
        seen += s
        edge.append(round(free * seen / total))
    rows = [0] * c["E"]
    for i, e in enumerate(who):
        rows[e] = 1 + edge[i + 1] - edge[i]
    return rows


def _codes(shape, group, zeros, g, std):
    """4-bit weights as a quantizer leaves them: bytes (even k in the low nibble), scales, zero points."""
    w = torch.randn(shape, generator=g, device=DEV).mul_(std).view(*shape[:-1], shape[-1] // (group or 32), group or 32)
    z = None
    if group == 0:  # MXFP4: E2M1 codes, one power of two per 32 values
        e = torch.floor(torch.log2(w.abs().amax(dim=-1).clamp_min(1e-30))) - 2.0
        w = w * torch.exp2(-e)[..., None]
        mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
        code = torch.bucketize(w.abs(), mids, out_int32=True).to(torch.uint8) + (w < 0).to(torch.uint8) * 8
        s = (e + 127.0).to(torch.uint8)
    elif zeros:
        lo, hi = w.amin(dim=-1).clamp_max(0.0), w.amax(dim=-1).clamp_min(0.0)
        s = ((hi - lo) / 15.0).to(BF16)
        z = torch.round(-lo / s.float()).clamp_(0.0, 15.0)
        code = (torch.round(w / s.float()[..., None]) + z[..., None]).clamp_(0.0, 15.0).to(torch.uint8)
        z = z.to(torch.uint8)
    else:
        s = (w.abs().amax(dim=-1) / 7.0).to(BF16)
        code = (torch.round(w / s.float()[..., None]).clamp_(-8.0, 7.0) + 8.0).to(torch.uint8)
    code = code.view(*shape)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), s, z


def _inputs(c, seed):
    k, g = c["kind"], _gen(seed)
    N, K = c["N"], c["K"]
    std = 1.0 / math.sqrt(K)  # projections of about unit variance
    if k == "w4_quant":
        return {"w": _randn((N, K), g, std)}
    if k == "w4":
        q, s, z = _codes((N, K), c["group"], c["zeros"], g, std)
        return {"x": _randn((c["M"], K), g), "q": q, "s": s, "z": z}
    E, M = c["E"], c["M"]
    rows = _counts(c, seed)
    offs = [0]
    for r in rows:
        offs.append(offs[-1] + r)
    d = {"rows": rows, "offs": torch.tensor(offs, dtype=torch.int32, device=DEV)}
    if k == "w4_grouped":
        q, s, z = _codes((E, N, K), c["group"], c["zeros"], g, std)
        tokens = M // c["topk"]
        gather = torch.randperm(M, generator=g, device=DEV).to(torch.int32)
        return {**d, "x": _randn((tokens, K), g), "q": q, "s": s, "z": z, "gather": gather}
    d.update(x=_randn((M, K), g), w=_randn((E, N, K), g, std))
    if k == "grouped_bwd":
        d["dy"] = _randn((M, N), g, 0.1)
    return d


def prepare(case, seed):
    """The state holds the outputs and workspaces that the library's calls write; the plain forms make their own."""
    c = case
    s = _inputs(c, seed)
    s["case"] = c
    k, N, K = c["kind"], c["N"], c["K"]

    def out(shape, dtype=BF16):
        return torch.empty(shape, dtype=dtype, device=DEV)

    if k == "w4_quant":
        s["q"], s["s"] = out((N, K // 2), torch.uint8), out((N, K // c["group"]))
        s["z"] = out((N, K // c["group"]), torch.uint8) if c["zeros"] else None
        s["back"] = out((N, K))
    elif k == "grouped_bwd":
        s["dx"], s["dw"] = out((c["M"], K)), out((c["E"], N, K))
    else:
        s["y"] = out((c["M"], N))
    if "rows" in s:
        s.update(_padding(s["rows"]))
    if own:
        s["call"], s["keep"] = _bind(s)
    return s


def _padding(rows):
    """The plain forms' plan of a batch: the experts that have rows, the [experts, most rows] table of their row
    numbers (the last row again where an expert has fewer) and each row's place in it."""
    who = [e for e, r in enumerate(rows) if r]
    most = max(rows)
    first, at = {}, 0
    for e, r in enumerate(rows):
        first[e] = at
        at += r
    table = [[first[e] + min(i, rows[e] - 1) for i in range(most)] for e in who]
    live = [[i < rows[e] for i in range(most)] for e in who]
    place = [n * most + i for n, e in enumerate(who) for i in range(rows[e])]
    return {"who": torch.tensor(who, device=DEV), "table": torch.tensor(table, device=DEV),
            "live": torch.tensor(live, device=DEV), "place": torch.tensor(place, device=DEV)}


# ---------------------------------------------------------------------------
# one pass through the library
# ---------------------------------------------------------------------------
def _bind(s):
    """The library's call with its arguments fixed, as a serving loop binds it, and the workspace that it holds."""
    pkg = os.path.join(os.getcwd(), "amd-kernels_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import hkq

    c, k = s["case"], s["case"]["kind"]
    N, K = c["N"], c["K"]
    st = torch.cuda.current_stream().cuda_stream

    def p(name):
        return s[name].data_ptr() if s.get(name) is not None else None

    if k == "w4_quant":
        grp = c["group"]
        quant = hkq.bind("hkq_w4_quant", p("w"), p("q"), p("s"), p("z"), N, K, K, K // 2, K // grp, grp, st)
        back = hkq.bind("hkq_w4_dequant", p("q"), p("s"), p("z"), p("back"), N, K, K // 2, K // grp, K, grp, st)

        def both():
            quant()
            back()

        return both, None
    if k.startswith("w4"):
        kind, grp = (hkq.W4_MXFP4, 32) if c["group"] == 0 else (hkq.W4_INT4, c["group"])
        sizes = (c["M"], N, K) if k == "w4" else (c["M"], c["E"], N, K)
        name = "hkq_gemm_w4a16" if k == "w4" else "hkq_grouped_gemm_w4a16"
        n = int(getattr(hkq.lib(), name + "_workspace")(*sizes))
        ws = torch.empty(n, dtype=torch.uint8, device=DEV) if n else None
        wp = ws.data_ptr() if n else None
        if k == "w4":
            return hkq.bind(name, p("x"), p("q"), p("s"), p("z"), p("y"), c["M"], N, K, K, K // 2, K // grp, N, grp, kind,
                            wp, n, st), ws
        return hkq.bind(name, p("x"), p("q"), p("s"), p("z"), p("y"), p("offs"), p("gather"), c["M"], s["x"].shape[0],
                        c["E"], N, K, c["topk"], K, K // 2, N * (K // 2), K // grp, N * (K // grp), N, grp, kind, wp, n,
                        st), ws
    M, E = c["M"], c["E"]
    if k == "grouped":
        return hkq.bind("hkq_grouped_gemm_bf16", p("x"), p("w"), p("y"), p("offs"), M, E, N, K, K, K, N * K, N, st), None
    return hkq.bind("hkq_grouped_gemm_backward", p("dy"), p("x"), p("w"), p("dx"), p("dw"), p("offs"), M, E, N, K, N, K, K,
                    N * K, K, K, N * K, st), None


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _widened(q, s, z):
    """The float32 weights that 4-bit codes stand for."""
    code = torch.stack((q & 15, q >> 4), dim=-1).view(*s.shape, -1)
    if s.dtype == torch.uint8:
        return (torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)[code.int()]
                * torch.exp2(s.float() - 127.0)[..., None]).flatten(-2)
    off = 8.0 if z is None else z.float()[..., None]
    return ((code.float() - off) * s.float()[..., None]).flatten(-2)


def _spread(s, t):
    """The rows of t by expert, padded: [experts with rows, most rows, columns] in float32."""
    return t[s["table"]].float()


def _plain(s):
    c, k = s["case"], s["case"]["kind"]
    if k == "w4_quant":
        w = s["w"].float().view(c["N"], -1, c["group"])
        if c["zeros"]:
            lo, hi = w.amin(dim=-1).clamp_max(0.0), w.amax(dim=-1).clamp_min(0.0)
            sc = (hi / 15.0 - lo / 15.0).to(BF16)
            inv = 1.0 / sc.float()
            z = torch.round(-lo * inv).clamp(0.0, 15.0)
            code = (torch.round(w * inv[..., None]) + z[..., None]).clamp(0.0, 15.0) - z[..., None]
            return (code * sc.float()[..., None]).to(BF16).flatten(-2), sc, z.to(torch.uint8)
        sc = (w.abs().amax(dim=-1) / 7.0).to(BF16)
        code = torch.round(w * (1.0 / sc.float())[..., None]).clamp(-8.0, 7.0)
        return (code * sc.float()[..., None]).to(BF16).flatten(-2), sc
    if k == "w4":
        return (s["x"].float() @ _widened(s["q"], s["s"], s["z"]).t()).to(BF16)
    if k == "w4_grouped":
        w = _widened(s["q"][s["who"]], s["s"][s["who"]], None if s["z"] is None else s["z"][s["who"]])
        x = s["x"][torch.div(s["gather"], c["topk"], rounding_mode="floor")]
        return torch.bmm(_spread(s, x), w.transpose(1, 2)).flatten(0, 1)[s["place"]].to(BF16)
    x = _spread(s, s["x"])
    w = s["w"][s["who"]].float()
    if k == "grouped":
        return torch.bmm(x, w.transpose(1, 2)).flatten(0, 1)[s["place"]].to(BF16)
    dy = _spread(s, s["dy"]) * s["live"][..., None]
    dx = torch.bmm(dy, w).flatten(0, 1)[s["place"]].to(BF16)
    dw = torch.zeros((c["E"], c["N"], c["K"]), dtype=BF16, device=DEV)
    dw[s["who"]] = torch.bmm(dy.transpose(1, 2), x).to(BF16)
    return dx, dw


def run(state):
    s = state
    if not own:
        return _plain(s)
    s["call"]()
    k = s["case"]["kind"]
    if k == "w4_quant":
        return (s["back"], s["s"]) if s["z"] is None else (s["back"], s["s"], s["z"])
    return (s["dx"], s["dw"]) if k == "grouped_bwd" else s["y"]


# ---------------------------------------------------------------------------
# necessary work, float64 results
# ---------------------------------------------------------------------------
def _weight_bytes(n, group, zeros):
    """n 4-bit weights with their scales and zero points."""
    return n // 2 + (n // 32 if group == 0 else n // group * (3 if zeros else 2))


def work(case):
    c, k = case, case["kind"]
    N, K = c["N"], c["K"]
    if k == "w4_quant":  # read, codes written and read back, values written
        return {"bytes": 4 * N * K + 2 * _weight_bytes(N * K, c["group"], c["zeros"]), "flops": 6.0 * N * K}
    M = c["M"]
    if k == "w4":
        return {"bytes": _weight_bytes(N * K, c["group"], c["zeros"]) + 2 * M * (N + K), "flops": 2.0 * M * N * K}
    A, idx = c["active"], 4 * (c["E"] + 1)
    if k == "w4_grouped":
        return {"bytes": _weight_bytes(A * N * K, c["group"], c["zeros"]) + 2 * M // c["topk"] * K + 2 * M * N + 4 * M + idx,
                "flops": 2.0 * M * N * K}
    if k == "grouped":
        return {"bytes": 2 * (A * N * K + M * K + M * N) + idx, "flops": 2.0 * M * N * K}
    return {"bytes": 2 * (A * N * K + c["E"] * N * K + 2 * M * K + M * N) + idx, "flops": 4.0 * M * N * K}


def _weights64(d, e=None):
    """float64 weights of expert e (of the only matrix) from its codes, column by column of the pairs."""
    q, s, z = (None if t is None else t if e is None else t[e] for t in (d["q"], d["s"], d["z"]))
    w = torch.empty((q.shape[0], 2 * q.shape[1]), dtype=torch.float64, device=DEV)
    grp = w.shape[1] // s.shape[1]
    for half in (0, 1):
        nib = torch.bitwise_right_shift(q, 4 * half).bitwise_and(15)
        if s.dtype == torch.uint8:
            mag, e1 = (nib & 1).double(), ((nib >> 1) & 3).double()
            v = torch.where(e1 > 0, (1.0 + 0.5 * mag) * torch.pow(2.0, e1 - 1.0), 0.5 * mag)
            w[:, half::2] = torch.where(nib >= 8, -v, v)
        else:
            w[:, half::2] = nib.double()
    w = w.view(w.shape[0], -1, grp)
    if s.dtype == torch.uint8:
        return (w * torch.pow(2.0, s.double() - 127.0).unsqueeze(2)).view(w.shape[0], -1)
    w -= 8.0 if z is None else z.double().unsqueeze(2)
    return (w * s.double().unsqueeze(2)).view(w.shape[0], -1)


def exact(case, seed):
    c, k = case, case["kind"]
    d = _inputs(c, seed)
    if k == "w4_quant":
        w = d["w"].double().view(c["N"], c["K"] // c["group"], c["group"])
        if c["zeros"]:
            low, top = torch.clamp(w.min(dim=2)[0], max=0.0), torch.clamp(w.max(dim=2)[0], min=0.0)
            s = ((top - low) / 15.0).float().to(BF16).double()
            z = torch.round(-low / s).clamp(0, 15)
            v = torch.clamp(torch.round(w / s.unsqueeze(2)) + z.unsqueeze(2), 0, 15) - z.unsqueeze(2)
            return (v * s.unsqueeze(2)).view(c["N"], -1), s, None
        s = (torch.linalg.vector_norm(w, ord=math.inf, dim=2) / 7.0).float().to(BF16).double()
        return (torch.clamp(torch.round(w / s.unsqueeze(2)), -8, 7) * s.unsqueeze(2)).view(c["N"], -1), s
    if k == "w4":
        return torch.mm(d["x"].double(), _weights64(d).t())
    M, N, K = c["M"], c["N"], c["K"]
    out = torch.empty((M, N), dtype=torch.float64, device=DEV)
    dx = torch.empty((M, K), dtype=torch.float64, device=DEV) if k == "grouped_bwd" else None
    dw = torch.zeros((c["E"], N, K), dtype=torch.float64, device=DEV) if k == "grouped_bwd" else None
    at = 0
    for e, r in enumerate(d["rows"]):
        rows = slice(at, at + r)
        at += r
        if not r:
            continue
        if k == "w4_grouped":
            out[rows] = torch.mm(d["x"][(d["gather"][rows] // c["topk"]).long()].double(), _weights64(d, e).t())
        elif k == "grouped":
            out[rows] = torch.mm(d["x"][rows].double(), d["w"][e].double().t())
        else:
            dy = d["dy"][rows].double()
            dx[rows] = torch.mm(dy, d["w"][e].double())
            dw[e] = torch.mm(dy.t(), d["x"][rows].double())
    return out if dx is None else (dx, dw)
