"""What layer norm, token log probabilities and the distillation loss refuse, through the C ABI: every call here
fails its checks before the device is touched.  And the definitions in 64 bits against torch's own."""
import math

import pytest

import motifcl_amd

from . import rows64

torch = pytest.importorskip("torch")
P = 0x100000  # a device address that is never used
F32, F16 = 0, 1
BIG = 1 << 62


@pytest.fixture(scope="module")
def L():
    return motifcl_amd.load()


def refused(L, rc, needle):
    assert rc == -1 and needle in L.mcc_last_error().decode(), L.mcc_last_error().decode()


def norm(L, x=P, xn=4 * 64, xs=16, gain=None, gn=0, bias=None, bn=0, y=2 * P, yn=4 * 64, ys=16, mean=None, mn=0,
         rstd=None, rn=0, rows=4, cols=16, element=F32, eps=1e-5):
    return L.mcc_layer_norm(None, x, xn, xs, gain, gn, bias, bn, y, yn, ys, mean, mn, rstd, rn, rows, cols, element, eps)


@pytest.mark.parametrize("kwargs, needle", [
    (dict(rows=0), "non-zero"), (dict(cols=0), "non-zero"), (dict(element=3), "element type"), (dict(element=-1), "element type"),
    (dict(cols=(1 << 30) + 1, xn=BIG, yn=BIG), "2^30"), (dict(rows=1 << 31, xn=BIG, yn=BIG), "rows exceed"),
    (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"),
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(x=P + 2), "aligned"), (dict(y=2 * P + 1), "aligned"),
    (dict(xs=15), "stride shorter"), (dict(ys=0), "stride shorter"), (dict(xs=BIG), "overflows"),
    (dict(xn=255), "x buffer is too small"), (dict(yn=255), "y buffer is too small"), (dict(xs=17), "x buffer is too small"),
    (dict(gain=P + 2, gn=64), "gain must be 4-byte"), (dict(gain=P, gn=63), "gain buffer is too small"),
    (dict(bias=P, bn=60), "bias buffer is too small"), (dict(mean=P, mn=15), "mean buffer is too small"),
    (dict(rstd=P, rn=0), "rstd buffer is too small"),
    (dict(y=P + 64), "y overlaps x"), (dict(y=P, ys=17, yn=400), "y overlaps x"),
    (dict(xs=24, xn=4 * 88, y=P + 40, ys=24, yn=4 * 88), "y overlaps x"),
])
def test_layer_norm_refuses(L, kwargs, needle):
    refused(L, norm(L, **kwargs), needle)


def norm_backward(L, d=P, dn=256, ds=16, x=2 * P, xn=256, xs=16, mean=3 * P, mn=16, rstd=4 * P, rn=16, gain=None, gn=0,
                  gx=5 * P, gxn=256, gxs=16, gg=None, ggn=0, gb=6 * P, gbn=64, ws=7 * P, wsn=BIG, rows=4, cols=16, element=F32):
    return L.mcc_layer_norm_backward(None, d, dn, ds, x, xn, xs, mean, mn, rstd, rn, gain, gn, gx, gxn, gxs, gg, ggn, gb,
                                     gbn, ws, wsn, rows, cols, element)


@pytest.mark.parametrize("kwargs, needle", [
    (dict(rows=0), "non-zero"), (dict(element=9), "element type"), (dict(d=None), "null"), (dict(x=None), "null"),
    (dict(mean=None), "null"), (dict(rstd=None), "null"), (dict(mn=12), "mean buffer"), (dict(rn=15), "rstd buffer"),
    (dict(dn=255), "grad_out buffer"), (dict(gx=P + 4), "grad_x overlaps grad_out"), (dict(gx=2 * P + 4), "grad_x overlaps x"),
    (dict(gx=P, gxs=32, gxn=4 * 112), "grad_x overlaps grad_out"), (dict(gb=6 * P, gbn=63), "grad_bias buffer"),
    (dict(gg=P, ggn=0), "grad_gain buffer"), (dict(gx=None, gb=None), "no output"),
    (dict(rows=40, dn=4 * 640, xn=4 * 640, gxn=4 * 640, mn=160, rn=160, ws=None), "null"),
    (dict(rows=40, dn=4 * 640, xn=4 * 640, gxn=4 * 640, mn=160, rn=160, ws=P + 8), "16-byte"),
    (dict(rows=40, dn=4 * 640, xn=4 * 640, gxn=4 * 640, mn=160, rn=160, wsn=64), "workspace is too small"),
])
def test_layer_norm_backward_refuses(L, kwargs, needle):
    refused(L, norm_backward(L, **kwargs), needle)


def log_probs(L, z=P, zn=4 * 400, zs=100, tok=2 * P, tokn=16, lp=3 * P, lpn=16, h=4 * P, hn=16, lse=5 * P, lsen=16,
              ids=6 * P, idsn=80, best=7 * P, bestn=80, ws=None, wsn=0, rows=4, vocab=100, top=5, element=F32, t=1.0):
    return L.mcc_token_log_probs(None, z, zn, zs, tok, tokn, lp, lpn, h, hn, lse, lsen, ids, idsn, best, bestn, ws, wsn,
                                 rows, vocab, top, element, t)


@pytest.mark.parametrize("kwargs, needle", [
    (dict(rows=0), "non-zero"), (dict(vocab=0), "non-zero"), (dict(element=7), "element type"),
    (dict(t=0.0), "temperature"), (dict(t=-1.0), "temperature"), (dict(t=math.nan), "temperature"),
    (dict(t=math.inf), "temperature"), (dict(t=1e-45), "temperature"),
    (dict(top=101), "alternatives"), (dict(top=129, vocab=1000, zs=1000, zn=16000), "alternatives"),
    (dict(z=None), "null"), (dict(z=P + 2), "aligned"), (dict(zs=99), "stride shorter"), (dict(zn=1599), "logits buffer"),
    (dict(tokn=15), "tokens buffer"), (dict(tok=P + 1), "tokens must be"), (dict(lpn=15), "log_prob buffer"),
    (dict(hn=15), "entropy buffer"), (dict(lsen=0), "lse buffer"), (dict(idsn=79), "top_ids buffer"),
    (dict(bestn=79), "top_log_probs buffer"),
    (dict(vocab=40000, zs=40000, zn=4 * 160000), "null"),
    (dict(vocab=40000, zs=40000, zn=4 * 160000, ws=P + 4, wsn=BIG), "16-byte"),
    (dict(vocab=40000, zs=40000, zn=4 * 160000, ws=P, wsn=100), "workspace is too small"),
])
def test_token_log_probs_refuses(L, kwargs, needle):
    refused(L, log_probs(L, **kwargs), needle)


def log_probs_backward(L, z=P, zn=1600, zs=100, tok=2 * P, tokn=16, lse=3 * P, lsen=16, h=4 * P, hn=16, up=5 * P, upn=16,
                       uph=None, uphn=0, out=6 * P, outn=1600, outs=100, rows=4, vocab=100, element=F32, t=1.0):
    return L.mcc_token_log_probs_backward(None, z, zn, zs, tok, tokn, lse, lsen, h, hn, up, upn, uph, uphn, out, outn,
                                          outs, rows, vocab, element, t)


@pytest.mark.parametrize("kwargs, needle", [
    (dict(rows=0), "non-zero"), (dict(t=0.0), "temperature"), (dict(z=None), "null"), (dict(out=None), "null"),
    (dict(tok=None), "null"), (dict(lse=None), "null"), (dict(up=None), "no upstream"),
    (dict(uph=P, uphn=16, h=None), "null"), (dict(uph=P, uphn=15), "grad_entropy buffer"), (dict(upn=12), "grad_log_prob buffer"),
    (dict(outn=1599), "grad_logits buffer"), (dict(outs=50), "stride shorter"), (dict(out=P + 400), "overlaps logits"),
])
def test_token_log_probs_backward_refuses(L, kwargs, needle):
    refused(L, log_probs_backward(L, **kwargs), needle)


def distill(L, z=P, zn=1600, zs=100, ids=2 * P, idsn=80, y=3 * P, yn=80, w=None, wn=0, loss=4 * P, lossn=16, out=5 * P,
            outn=1600, outs=100, rows=4, vocab=100, top=5, element=F32, t=1.0):
    return L.mcc_distill_top(None, z, zn, zs, ids, idsn, y, yn, w, wn, loss, lossn, out, outn, outs, rows, vocab, top,
                             element, t)


@pytest.mark.parametrize("kwargs, needle", [
    (dict(vocab=0), "non-zero"), (dict(top=0), "1 to 128"), (dict(top=129, idsn=BIG, yn=BIG), "1 to 128"),
    (dict(t=-2.0), "temperature"), (dict(t=1e30), "square"), (dict(z=None), "null"), (dict(ids=None), "null"), (dict(y=None), "null"),
    (dict(idsn=79), "teacher_ids buffer"), (dict(yn=79), "teacher_logits buffer"), (dict(w=P, wn=15), "weight buffer"),
    (dict(lossn=15), "loss buffer"), (dict(loss=None, out=None), "no output"), (dict(outn=100), "grad_logits buffer"),
    (dict(out=P + 4), "overlaps logits"),
])
def test_distill_top_refuses(L, kwargs, needle):
    refused(L, distill(L, **kwargs), needle)


def test_workspace_sizes(L):
    assert L.mcc_token_log_probs_workspace_nbytes(4, 100, 5, F32) == 0
    assert L.mcc_token_log_probs_workspace_nbytes(4, 40000, 5, F32) > 0
    assert L.mcc_token_log_probs_workspace_nbytes(4, 40000, 129, F32) == 0
    assert L.mcc_token_log_probs_workspace_nbytes(0, 40000, 5, F32) == 0
    assert L.mcc_layer_norm_backward_workspace_nbytes(1, 64, F32) == 0
    assert L.mcc_layer_norm_backward_workspace_nbytes(1000, 64, F16) > 0


def test_definitions_agree_with_torch():
    g = torch.Generator().manual_seed(2)
    x, dy = (torch.randn(4, 33, generator=g, dtype=torch.float64) for _ in range(2))
    gain, bias = (torch.randn(33, generator=g, dtype=torch.float64) for _ in range(2))
    leaves = [t.clone().requires_grad_() for t in (x, gain, bias)]
    y = torch.nn.functional.layer_norm(leaves[0], (33,), leaves[1], leaves[2], 1e-5)
    want = torch.autograd.grad(y, leaves, dy)
    got, mean, rstd = rows64.layer_norm(x, gain, bias, 1e-5)
    assert torch.allclose(got, y)
    for a, b in zip(rows64.layer_norm_backward(dy, x, mean, rstd, gain), want):
        assert torch.allclose(a, b)
    z = x.clone().requires_grad_()
    tokens, t = torch.tensor([3, -1, 40, 32], dtype=torch.int32), 0.7
    up, up_h = torch.randn(4, generator=g, dtype=torch.float64), torch.randn(4, generator=g, dtype=torch.float64)
    log_p = torch.log_softmax(z / t, 1)
    h = torch.distributions.Categorical(logits=z / t).entropy()
    picked = torch.stack([log_p[0, 3], 0 * z[1, 0], 0 * z[2, 0], log_p[3, 32]])
    got = rows64.token_log_probs(x, tokens, t)
    assert torch.allclose(got[0], picked) and torch.allclose(got[1], h) and torch.allclose(got[2], torch.logsumexp(z / t, 1))
    want, = torch.autograd.grad((picked * up + h * up_h).sum(), z, retain_graph=True)
    assert torch.allclose(rows64.token_log_probs_backward(x, tokens, up, up_h, t)[0], want)
    ids = torch.tensor([[3, 3], [0, -1], [32, 5], [-1, 33]], dtype=torch.int32)
    y = torch.randn(4, 2, generator=g, dtype=torch.float64)
    loss, grad, _, _ = rows64.distill_top(x, ids, y, up, t)
    q = [torch.softmax(y[0] / t, 0), torch.ones(1, dtype=torch.float64), torch.softmax(y[2] / t, 0)]
    rows = [(q[0] * (q[0].log() - log_p[0, [3, 3]])).sum(), -log_p[1, 0], (q[2] * (q[2].log() - log_p[2, [32, 5]])).sum()]
    rows = t * t * torch.stack(rows + [0 * z[3, 0]])
    assert torch.allclose(loss, rows)
    assert torch.allclose(grad, torch.autograd.grad((rows * up).sum(), z)[0])
    assert rows64.top_ids(torch.tensor([[0.0, math.nan, -0.0, -math.inf, 2.0]]), 5).tolist() == [[4, 0, 2, 3, 1]]
