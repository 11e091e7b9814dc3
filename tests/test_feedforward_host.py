"""Host-side checks of the feed-forward operators (no GPU needed): what their C
entry points and their tensor layer refuse before any launch, and the
workspace query."""
import pytest
import torch

import hkq

P = 0x1000  # never dereferenced: validation fails first
BF16 = torch.bfloat16


def refused(name, *args, match):
    with pytest.raises(hkq.HkqError, match=match) as e:
        hkq.call(name, *args)
    assert "code 1" in str(e.value)


def norm(**kw):
    a = dict(x=P, res=P, w=P, h=P, q=P, s=P, M=4, D=256, ldx=256, ldr=256, ldh=256, ldq=256, lds=2, eps=1e-6, group=128,
             kind=0)
    a.update(kw)
    return ("hkq_add_rmsnorm_quant", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(kind=2), "kind"), (dict(group=64), "group"), (dict(M=-1), "M must"), (dict(M=1 << 31), "M must"), (dict(M=1 << 26), "M must"),
    (dict(M=1 << 24, D=2176, ldx=2176, ldr=2176, ldh=2176, ldq=2176, lds=17), "M must"),
    (dict(D=260, ldx=264), "multiple of 8"), (dict(D=4, group=0), "multiple of 8"), (dict(D=16392, group=0), "16384"),
    (dict(D=200), "128 with groups"), (dict(ldx=248), "ldx"), (dict(ldx=260), "ldx"), (dict(ldr=100), "ldr"),
    (dict(ldh=252), "ldh"), (dict(ldq=260), "ldq"), (dict(lds=1), "lds"), (dict(eps=-1.0), "eps"),
    (dict(h=P, res=2 * P, ldh=264), "pitch"), (dict(x=2 * P, h=P, ldh=264), "pitch"), (dict(h=None), "both or neither"), (dict(res=None), "both or neither"), (dict(w=None), "required"),
    (dict(x=P + 8), "aligned"), (dict(res=P + 8), "aligned"), (dict(h=P + 2), "aligned"), (dict(q=P + 4), "aligned")])
def test_norm_refusals(kw, match):
    refused(*norm(**kw), match=match)


def epilogue(kind, **kw):
    fp8 = kind == "a8w8"
    a = dict(A=P, B=P, **(dict(sa=P, sb=P) if fp8 else {}), bias=P, res=P, C=2 * P, M=16, N=64, K=128, lda=128, ldb=128,
             ldr=64, ldc=64, act=2, alpha=1.0, ws=None, n=0)
    a.update(kw)
    return (f"hkq_gemm_{kind}_epilogue", *a.values(), None)


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("kw,match", [
    (dict(M=-1), "M, N must"), (dict(N=62), "N must be a multiple of 4"), (dict(K=0), "K > 0"), (dict(K=40, lda=48, ldb=48), "K must be"),
    (dict(M=1 << 30), "2\\^30"), (dict(lda=64), "lda"), (dict(ldb=132), "ldb"), (dict(ldc=60), "ldc"), (dict(ldc=66), "ldc"),
    (dict(ldr=60), "ldr"), (dict(ldr=66), "ldr"), (dict(act=5), "act"), (dict(act=-1), "act"),
    (dict(alpha=float("nan")), "alpha"), (dict(alpha=float("inf")), "alpha"), (dict(alpha=2e30), "alpha"), (dict(res=2 * P, ldr=128), "pitch"),
    (dict(ldc=1 << 24), "ldc"), (dict(ldr=1 << 24), "ldr"),
    (dict(A=None), "required"), (dict(C=None), "required"), (dict(A=P + 8), "aligned"), (dict(B=P + 4), "aligned"),
    (dict(C=2 * P + 4), "aligned"), (dict(bias=P + 4), "aligned"), (dict(res=P + 2), "aligned"), (dict(ws=P + 4, n=64), "aligned"),
    (dict(lda=1 << 27, ldb=1 << 27), "row pitches too large")])
def test_epilogue_refusals(kind, kw, match):
    refused(*epilogue(kind, **kw), match=match)


def gated(kind, **kw):
    fp8 = kind == "a8w8"
    a = dict(X=P, W=P, **(dict(sx=P, sw=P) if fp8 else {}), H=P, **({} if fp8 else dict(Y=P)), M=16, F=64, K=128, ldx=128,
             ldw=128, ldh=64, **({} if fp8 else dict(ldy=128)), act=2, alpha=1.0, inter=0)
    a.update(kw)
    return (f"hkq_gated_ffn_{kind}", *a.values(), None)


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("kw,match", [
    (dict(M=-1), "M, F must"), (dict(F=60), "multiple of 8"), (dict(F=1 << 28), "2\\^28"), (dict(K=40, ldx=48, ldw=48), "K must be"),
    (dict(ldx=64), "ldx"), (dict(ldw=132), "ldw"), (dict(ldh=60), "ldh"), (dict(ldh=1 << 24), "ldh"), (dict(act=9), "act"), (dict(alpha=float("inf")), "alpha"),
    (dict(W=None), "required"), (dict(X=P + 8), "aligned"), (dict(H=P + 4), "aligned"),
    (dict(ldw=1 << 27), "row pitches too large"), (dict(ldw=1 << 26, inter=1), "row pitches too large")])
def test_gated_refusals(kind, kw, match):
    refused(*gated(kind, **kw), match=match)


def test_gated_kept_projections_refusals():
    refused(*gated("bf16", ldy=120), match="ldy")
    refused(*gated("bf16", ldy=130), match="ldy")
    refused(*gated("bf16", Y=P + 4), match="aligned")


def backward(**kw):
    a = dict(dH=P, X=P, W=P, Y=P, dX=P, dW=P, M=16, F=64, K=128, lddh=64, ldx=128, ldw=128, ldy=128, lddx=128, lddw=128,
             act=2, alpha=1.0, inter=0, ws=P, n=1 << 30)
    a.update(kw)
    return ("hkq_gated_ffn_backward", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(M=-1), "M, F must"), (dict(M=1 << 29), "2\\^29"), (dict(F=60), "multiple of 8"), (dict(F=(1 << 20) + 8), "2\\^20"), (dict(K=48), "multiple of 32"),
    (dict(lddh=60), "lddh"), (dict(ldx=100), "ldx"), (dict(ldw=132), "ldw"), (dict(ldx=1 << 24), "ldx"), (dict(ldy=132), "ldy"),
    (dict(lddx=100), "lddx"), (dict(lddw=130), "lddw"), (dict(lddx=1 << 23), "lddx"), (dict(lddw=1 << 23), "lddw"), (dict(act=5), "act"), (dict(alpha=float("nan")), "alpha"),
    (dict(dH=None), "required"), (dict(X=None), "required"), (dict(W=None), "required"), (dict(n=0), "workspace"),
    (dict(ws=None), "workspace"), (dict(ws=P + 8), "aligned"), (dict(Y=P + 8), "aligned"), (dict(dX=P + 4), "aligned")])
def test_backward_refusals(kw, match):
    refused(*backward(**kw), match=match)


def test_backward_workspace_query():
    """The projections' gradients, and split sums where a product has few tiles."""
    q = hkq.lib().hkq_gated_ffn_backward_workspace
    assert q(0, 64, 64) == q(4, 0, 64) == q(-1, 64, 64) == 0
    assert q(4096, 14336, 4096) == 4096 * 28672 * 2          # many tiles each: no split
    assert q(10, 40, 64) == 10 * 128 * 2                     # rows of whole 64-value K-tiles
    assert q(16, 14336, 512) > 16 * 28672 * 2                # 4 tiles over 448 K-tiles
    # dX's 64 tiles of 256 x 256 in four parts
    assert q(1024, 14336, 4096) == 4096 + 4 * 64 * 256 * 256 * 4 + 1024 * 28672 * 2


def test_tensor_layer_refusals():
    """Shapes, types and names are checked before the library is asked (host tensors suffice)."""
    x, w = torch.zeros(4, 64, dtype=BF16), torch.zeros(32, 64, dtype=BF16)
    with pytest.raises(ValueError, match="act must be one of"):
        hkq.gemm_bf16_epilogue(x, w, act="swish")
    with pytest.raises(ValueError, match="B must be"):
        hkq.gemm_bf16_epilogue(x, torch.zeros(32, 60, dtype=BF16))
    with pytest.raises(TypeError, match="A has dtype"):
        hkq.gemm_bf16_epilogue(x.float(), w)
    with pytest.raises(TypeError, match="A has dtype"):
        hkq.gemm_a8w8_epilogue(x, w, torch.zeros(4), torch.zeros(32))
    with pytest.raises(ValueError, match="bias must be"):
        hkq.gemm_bf16_epilogue(x, w, bias=torch.zeros(31, dtype=BF16))
    with pytest.raises(ValueError, match="residual must be"):
        hkq.gemm_bf16_epilogue(x, w, residual=torch.zeros(4, 31, dtype=BF16))
    with pytest.raises(ValueError, match="contiguous last dimension"):
        hkq.gemm_bf16_epilogue(torch.zeros(64, 4, dtype=BF16).t(), w)
    with pytest.raises(ValueError, match="W must be"):
        hkq.gated_ffn_bf16(x, torch.zeros(31, 64, dtype=BF16))
    with pytest.raises(ValueError, match="Y must be"):
        hkq.gated_ffn_bf16(x, w, Y=torch.zeros(4, 16, dtype=BF16))
    with pytest.raises(TypeError, match="sw has dtype"):
        hkq.gated_ffn_a8w8(x.view(torch.uint8)[:, :64], w.view(torch.uint8)[:, :64], torch.zeros(4), torch.zeros(32, dtype=BF16))
    with pytest.raises(ValueError, match="dH must be"):
        hkq.gated_ffn_backward(torch.zeros(4, 8, dtype=BF16), x, w, torch.zeros(4, 32, dtype=BF16))
    with pytest.raises(ValueError, match="w must be"):
        hkq.add_rmsnorm_quant(x, torch.zeros(32, dtype=BF16))
    with pytest.raises(ValueError, match="h is written with a residual only"):
        hkq.add_rmsnorm_quant(x, torch.zeros(64, dtype=BF16), h=x)
    with pytest.raises(TypeError, match="q has dtype"):
        hkq.add_rmsnorm_quant(x, torch.zeros(64, dtype=BF16), kind=hkq.KIND_INT8, q=torch.zeros(4, 64, dtype=torch.uint8))


def test_modules_offer_the_operators():
    import hipkittens as hk

    x = torch.zeros(4, 64, dtype=BF16)
    for name in ("fused_gemm_a8w8_epilogue_tk", "fused_gemm_a16w16_epilogue_tk", "gated_ffn_tk"):
        assert name in hk.modules
    with pytest.raises(ValueError, match="GPU tensor"):
        hk.fused_gemm.a16w16_epilogue.dispatch(x, x, x)
    with pytest.raises(ValueError, match="GPU tensor"):
        hk.ffn.gated.gated_ffn_bf16(x, x, x)
    with pytest.raises(ValueError, match="GPU tensor"):
        hk.fused_add_rmsnorm_quant_fwd(x, None, x, None, x, x, 1e-6)


@pytest.mark.parametrize("M", [(1 << 26) - 3, (1 << 26) - 1])
def test_norm_rows_of_one_launch(M):
    """Four rows per workgroup of 256 threads: 2^26 - 3 rows round up to 2^24 workgroups, 2^32 threads."""
    refused(*norm(M=M, D=8, ldx=8, ldr=8, ldh=8, ldq=8, lds=1, group=0), match="M must")


def places(**kw):
    """A backward call whose operands lie 1 MiB apart but for those given."""
    at = {n: (i + 1) << 20 for i, n in enumerate(("dH", "X", "W", "Y", "dX", "dW", "ws"))}
    return backward(**{**at, "n": 1 << 19, **kw})


MB = 1 << 20


@pytest.mark.parametrize("kw,match", [
    (dict(dX=3 * MB), "dX must not overlap W"), (dict(dX=3 * MB + 128 * 127 * 2 + 128), "dX must not overlap W"),
    (dict(dW=2 * MB), "dW must not overlap X"), (dict(dW=2 * MB, dX=2 * MB), "dW must not overlap X"),
    (dict(dX=6 * MB), "dX and dW must not overlap"), (dict(dX=2 * MB, dW=3 * MB), "dX over X and dW over W"),
    (dict(dX=7 * MB), "workspace"), (dict(dW=7 * MB - 64), "workspace"), (dict(X=7 * MB + 2048), "workspace"),
    # rows of one pitch: columns that meet by their last and first four; rows of two pitches
    (dict(dX=3 * MB + 248, lddx=256, ldw=256), "dX must not overlap W"),
    (dict(dX=3 * MB + 264, lddx=260, ldw=256), "dX must not overlap W")])
def test_backward_overlap_refusals(kw, match):
    refused(*places(**kw), match=match)


def test_backward_of_neither_gradient():
    """Nothing to compute: no workspace, no operand, no launch."""
    hkq.call(*backward(dX=None, dW=None, ws=None, n=0))
    hkq.call(*backward(dX=None, dW=None, ws=None, n=0, dH=None, X=None, W=None, Y=None))
    refused(*backward(dX=None, dW=None, ws=None, n=0, act=5), match="act")


def apart(names):
    """Operands 1 MiB apart, in order."""
    return {n: (i + 1) << 20 for i, n in enumerate(names)}


NORM = apart(("x", "res", "w", "h", "q", "s"))


@pytest.mark.parametrize("kw,match", [
    (dict(h=NORM["x"] + 512), "h must be x or res"), (dict(h=NORM["res"] + 16), "h must be x or res"), (dict(h=NORM["w"]), "h must"),
    (dict(q=NORM["x"]), "q must not"), (dict(q=NORM["res"] + 64), "q must not"), (dict(q=NORM["w"]), "q must not"),
    (dict(q=NORM["h"]), "q must not"), (dict(s=NORM["x"] + 2032), "s must not"), (dict(s=NORM["w"]), "s must not"),
    (dict(s=NORM["h"]), "s must not"), (dict(s=NORM["q"] + 1020), "s must not"), (dict(s=NORM["q"], group=0, lds=1), "s must not"),
    (dict(q=NORM["x"], res=None, h=None), "q must not")])
def test_norm_overlap_refusals(kw, match):
    refused(*norm(**{**NORM, **kw}), match=match)


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("kw,match", [
    (dict(C="A"), "C must not"), (dict(C="B"), "C must not"), (dict(C="bias"), "C must not"), (dict(C="res", off=128), "C itself"),
    (dict(C="res", off=64), "C itself"), (dict(C="sa"), "C must not"), (dict(C="sb"), "C must not"), (dict(C="ws"), "workspace"),
    (dict(C="res", off=-8), "C itself"), (dict(C="A", off=-128, ldc=128), "C must not")])
def test_epilogue_overlap_refusals(kind, kw, match):
    names = ("A", "B", *(("sa", "sb") if kind == "a8w8" else ()), "bias", "res", "C", "ws")
    at = apart(names)
    if kw["C"] not in at:
        return  # bf16 has no scales
    # 128 x 1024 x 8192: K split over workgroups, with a workspace in use
    big = dict(M=128, N=1024, K=8192, lda=8192, ldb=8192, ldr=1024, ldc=1024) if kw["C"] == "ws" else {}
    n = int(getattr(hkq.lib(), f"hkq_gemm_{kind}_workspace")(128, 1024, 8192))
    at = {k: v * 64 for k, v in at.items()} if big else at
    more = {k: v for k, v in kw.items() if k not in ("C", "off")}
    refused(*epilogue(kind, **{**at, "n": n, **big, "C": at[kw["C"]] + kw.get("off", 0), **more}), match=match)


@pytest.mark.parametrize("kind", ["a8w8", "bf16"])
@pytest.mark.parametrize("kw,match", [
    (dict(H="X"), "H must not"), (dict(H="W"), "H must not"), (dict(H="W", off=64 * 128), "H must not"), (dict(H="sx"), "H must not"),
    (dict(H="sw"), "H must not"), (dict(Y="X"), "Y must not"), (dict(Y="W"), "Y must not"), (dict(Y="H"), "Y must not"),
    (dict(Y="H", off=64, ldy=256, ldh=256), "Y must not")])
def test_gated_overlap_refusals(kind, kw, match):
    at = apart(("X", "W", *(("sx", "sw", "H") if kind == "a8w8" else ("H", "Y"))))
    (out, over), more = list(kw.items())[0], {k: v for k, v in kw.items() if k.startswith("ld")}
    if out not in at or over not in at:
        return  # FP8 keeps no projections, bf16 has no scales
    refused(*gated(kind, **{**at, out: at[over] + kw.get("off", 0), **more}), match=match)
