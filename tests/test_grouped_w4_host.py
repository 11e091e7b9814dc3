"""Host-side checks of the grouped products and the 4-bit weights (no GPU needed): what
their C entry points and their tensor layer refuse before any launch, and calls with
nothing to do."""
import pytest
import torch

import hkq

P = 0x1000  # never dereferenced: validation fails first
FAR = 1 << 40
BF16 = torch.bfloat16


def refused(name, *args, match):
    with pytest.raises(hkq.HkqError, match=match) as e:
        hkq.call(name, *args)
    assert "code 1" in str(e.value)


def fwd(**kw):
    a = dict(X=P, W=FAR, Y=2 * FAR, offs=3 * FAR, M=64, E=4, N=128, K=256, ldx=256, ldw=256, se=128 * 256, ldy=128)
    a.update(kw)
    return ("hkq_grouped_gemm_bf16", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(M=-1), ">= 0"), (dict(E=-1), ">= 0"), (dict(M=1 << 28), "2\\^28"), (dict(E=1 << 16), "2\\^16"), (dict(N=1 << 22, ldy=1 << 22), "2\\^22"),
    (dict(N=132, ldy=136), "multiples of 8"), (dict(K=252, ldx=256), "multiples of 8"), (dict(ldx=248), "ldx"), (dict(ldx=260), "ldx"),
    (dict(ldw=128), "ldw"), (dict(ldw=1 << 22), "ldw"), (dict(ldy=120), "ldy"), (dict(se=-8), "stride_we"), (dict(se=12), "stride_we"),
    (dict(X=None), "required"), (dict(W=None), "required"), (dict(Y=None), "required"), (dict(offs=None), "required"),
    (dict(X=P + 8), "aligned"), (dict(W=FAR + 2), "aligned"), (dict(Y=2 * FAR + 8), "aligned"), (dict(offs=3 * FAR + 2), "aligned"),
    (dict(Y=P), "overlap"), (dict(Y=FAR + 4 * 128 * 256 * 2 - 16), "overlap"), (dict(Y=3 * FAR), "overlap"),
    (dict(Y=P + 256, ldx=512, ldy=512), "overlap")])
def test_grouped_refusals(kw, match):
    refused(*fwd(**kw), match=match)


def bwd(**kw):
    a = dict(dY=P, X=FAR, W=2 * FAR, dX=3 * FAR, dW=4 * FAR, offs=5 * FAR, M=64, E=4, N=128, K=256, lddy=128, ldx=256, ldw=256,
             se=128 * 256, lddx=256, lddw=256, sd=128 * 256)
    a.update(kw)
    return ("hkq_grouped_gemm_backward", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(M=-1), ">= 0"), (dict(N=124, lddy=128), "multiples of 8"), (dict(lddy=64), "lddy"), (dict(ldx=64), "ldx"), (dict(ldw=64), "ldw"),
    (dict(lddx=64), "lddx"), (dict(lddw=64), "lddw"), (dict(lddw=260), "lddw"), (dict(se=4), "stride_we"), (dict(sd=4), "stride_dwe"),
    (dict(sd=64 * 256), "groups of dW"), (dict(sd=0), "groups of dW"), (dict(sd=256, lddw=512), "groups of dW"),
    (dict(dY=None), "required"), (dict(X=None), "required"), (dict(W=None), "required"), (dict(offs=None), "offs"),
    (dict(dY=P + 8), "aligned"), (dict(dX=3 * FAR + 8), "aligned"), (dict(dW=4 * FAR + 8), "aligned"),
    (dict(dX=P), "dX must"), (dict(dX=FAR), "dX must"), (dict(dX=2 * FAR), "dX must"), (dict(dX=5 * FAR), "dX must"),
    (dict(dW=P), "dW must"), (dict(dW=FAR), "dW must"), (dict(dW=2 * FAR), "dW must"), (dict(dW=3 * FAR), "dW must")])
def test_grouped_backward_refusals(kw, match):
    refused(*bwd(**kw), match=match)


@pytest.mark.parametrize("args", [fwd(M=0), fwd(E=0, offs=None), fwd(N=0, ldy=0, W=None), bwd(dX=None, dW=None), bwd(E=0, offs=None),
                                  bwd(K=0, dX=None, dW=None), bwd(M=0, dW=None)])
def test_grouped_nothing_to_do(args):
    hkq.call(*args)


def quant(**kw):
    a = dict(w=P, q=FAR, s=2 * FAR, z=3 * FAR, N=64, K=256, ldw=256, ldq=128, lds=2, group=128)
    a.update(kw)
    return ("hkq_w4_quant", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(N=-1), ">= 0"), (dict(N=1 << 22), "2\\^22"), (dict(group=16), "group"), (dict(group=256), "group"), (dict(K=192, ldw=192), "multiple of group"),
    (dict(ldw=128), "ldw"), (dict(ldw=260), "ldw"), (dict(ldq=64), "ldq"), (dict(ldq=130), "ldq"), (dict(lds=1), "lds"),
    (dict(w=None), "required"), (dict(q=None), "required"), (dict(s=None), "required"), (dict(w=P + 8), "aligned"), (dict(q=FAR + 2), "aligned"),
    (dict(s=2 * FAR + 1), "aligned"), (dict(q=P), "overlap"), (dict(s=P), "overlap"), (dict(z=2 * FAR), "overlap"), (dict(z=FAR), "overlap")])
def test_w4_quant_refusals(kw, match):
    refused(*quant(**kw), match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(out=None), "required"), (dict(out=FAR + 8), "aligned"), (dict(out=P), "overlap"), (dict(ldo=128), "ldo"), (dict(ldo=260), "ldo"),
    (dict(group=48), "group"), (dict(ldq=6), "ldq")])
def test_w4_dequant_refusals(kw, match):
    a = dict(q=P, s=2 * FAR, z=None, out=FAR, N=64, K=256, ldq=128, lds=2, ldo=256, group=128)
    a.update(kw)
    refused("hkq_w4_dequant", *a.values(), None, match=match)


def product(grouped, **kw):
    a = dict(X=P, Q=FAR, S=2 * FAR, Z=3 * FAR, C=4 * FAR)
    if grouped:
        a.update(offs=5 * FAR, gather=6 * FAR, M=64, T=32, E=4, N=128, K=256, topk=2, ldx=256, ldq=128, sq=128 * 128, lds=2,
                 ss=256, ldc=128, group=128, kind=0, ws=None, n=0)
    else:
        a.update(M=64, N=128, K=256, ldx=256, ldq=128, lds=2, ldc=128, group=128, kind=0, ws=None, n=0)
    a.update(kw)
    return ("hkq_grouped_gemm_w4a16" if grouped else "hkq_gemm_w4a16", *a.values(), None)


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("kw,match", [
    (dict(M=-1), ">= 0"), (dict(M=1 << 28), "2\\^28"), (dict(kind=2), "kind"), (dict(kind=1), "MXFP4"), (dict(kind=1, group=32, lds=8), "MXFP4"),
    (dict(group=96), "group"), (dict(K=320, ldx=320, ldq=160, lds=3), "multiple of group"), (dict(ldx=128), "ldx"), (dict(ldx=260), "ldx"),
    (dict(ldq=136), "ldq"), (dict(ldq=64), "ldq"), (dict(lds=1), "lds"), (dict(ldc=64), "ldc"), (dict(ldc=1 << 22), "ldc"),
    (dict(X=None), "required"), (dict(Q=None), "required"), (dict(S=None), "required"), (dict(C=None), "required"),
    (dict(X=P + 8), "aligned"), (dict(Q=FAR + 8), "aligned"), (dict(S=2 * FAR + 1), "aligned"), (dict(C=4 * FAR + 1), "aligned"),
    (dict(C=P), "overlap"), (dict(C=FAR), "overlap"), (dict(C=2 * FAR), "overlap"), (dict(C=3 * FAR), "overlap")])
def test_w4_product_refusals(grouped, kw, match):
    refused(*product(grouped, **kw), match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(E=1 << 16), "2\\^16"), (dict(T=-1), ">= 0"), (dict(topk=0), "topk"), (dict(topk=1 << 16), "topk"), (dict(sq=8), "stride_q"),
    (dict(ss=-1), "stride_s"), (dict(offs=None), "offs"), (dict(gather=None), "M rows"), (dict(T=1 << 22, ldx=256), "2\\^31"),
    (dict(offs=5 * FAR + 2), "aligned"), (dict(gather=6 * FAR + 2), "aligned"), (dict(C=5 * FAR), "overlap"), (dict(C=6 * FAR), "overlap")])
def test_w4_grouped_refusals(kw, match):
    refused(*product(True, **kw), match=match)


def test_w4_nothing_to_do():
    hkq.call(*quant(N=0))
    hkq.call(*quant(K=0, ldw=0, ldq=0, lds=0))
    for args in (product(False, M=0), product(False, N=0, ldc=0), product(True, M=0), product(True, E=0)):
        hkq.call(*args)


def test_tensor_layer_refusals():
    X, W = torch.zeros((8, 64), dtype=BF16), torch.zeros((2, 16, 64), dtype=BF16)
    offs = torch.zeros(3, dtype=torch.int32)
    Y = torch.zeros((8, 16), dtype=BF16)
    for args, err, match in [((X, W, offs[:2]), ValueError, "offs"), ((X, W, offs.long()), TypeError, "offs"),
                             ((X[:, :32], W, offs), ValueError, "W"), ((X.float(), W, offs), TypeError, "X"),
                             ((X, W, offs, Y[:, :8]), ValueError, "Y"), ((X, W.transpose(1, 2), offs), ValueError, "W")]:
        with pytest.raises(err, match=match):
            hkq.grouped_gemm_bf16(*args)
    for kw, err, match in [(dict(dY=Y[:4]), ValueError, "dY"), (dict(dX=Y), ValueError, "dX"), (dict(dW=W[:1]), ValueError, "dW"),
                           (dict(dW=W.float()), TypeError, "dW")]:
        a = dict(dY=Y, X=X, W=W, offs=offs)
        a.update(kw)
        with pytest.raises(err, match=match):
            hkq.grouped_gemm_backward(**a)
    q, s, z = torch.zeros((16, 32), dtype=torch.uint8), torch.zeros((16, 2), dtype=BF16), torch.zeros((16, 2), dtype=torch.uint8)
    for args, err, match in [((X, q[:, :16], s), ValueError, "Q"), ((X, q.float(), s), TypeError, "Q"), ((X, q, s[:, :1].float()), TypeError, "S"),
                             ((X, q, s[:8]), ValueError, "S"), ((X, q, torch.zeros((16, 3), dtype=BF16)), ValueError, "groups"),
                             ((X, q, s, z[:, :1]), ValueError, "Z"), ((X, q, s, torch.zeros((16, 4), dtype=torch.uint8)[:, :2]), ValueError, "strides"),
                             ((X, q, z, z), ValueError, "zero points"), ((X, q, s, z, Y[:, :8]), ValueError, "C"),
                             ((X, q, s, z.float()), TypeError, "Z")]:
        with pytest.raises(err, match=match):
            hkq.gemm_w4a16(*args)
    Q, S = q[None].repeat(2, 1, 1), s[None].repeat(2, 1, 1)
    for kw, err, match in [(dict(offs=offs[:2]), ValueError, "offs"), (dict(gather=torch.zeros(4)), TypeError, "gather"),
                           (dict(S=s), ValueError, "scales"), (dict(Y=Y[:3]), ValueError, "Y")]:
        a = dict(X=X, Q=Q, S=S, offs=offs)
        a.update(kw)
        with pytest.raises(err, match=match):
            hkq.grouped_gemm_w4a16(**a)
    with pytest.raises(ValueError, match="group"):
        hkq.w4_quant(X, 48)
    with pytest.raises(ValueError, match="multiple of 128"):
        hkq.w4_quant(X, 128)
    with pytest.raises(TypeError, match="dtype"):
        hkq.w4_quant(X.float(), 32)
    with pytest.raises(TypeError, match="bf16"):
        hkq.w4_dequant(q, z)


def test_modules_are_found_and_refuse_host_tensors():
    import hipkittens as hk

    for name in ("grouped_gemm_tk", "w4_tk"):
        assert name in hk.modules, name
    X, W, offs = torch.zeros((8, 64), dtype=BF16), torch.zeros((2, 16, 64), dtype=BF16), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        hk.moe.grouped.grouped_gemm_bf16(X, W, X, offs)
    with pytest.raises(ValueError, match="GPU tensor"):
        hk.w4.gemm_w4a16(X, X, X, X)
