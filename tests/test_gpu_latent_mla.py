"""Dense latent attention (LatentMLA, LatentMLAExpanded) against 64-bit results, with the
bounds that oracle/latent_mla.py derives from the kernels' roundings."""
import pytest
import torch

from cppmega_amd import latent_mla_ops as ops
from oracle import latent_mla as orc

pytestmark = pytest.mark.gpu


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16)


def _docs(gen, B, S):
    """Packed documents of random lengths with padding (empty rows) behind the last."""
    starts, ends = torch.zeros(B, S, dtype=torch.int32), torch.zeros(B, S, dtype=torch.int32)
    for b in range(B):
        at, stop = 0, S - S // 7
        while at < stop:
            n = min(int(torch.randint(1, max(2, S // 3) + 1, (1,), generator=gen)), stop - at)
            starts[b, at:at + n] = at
            ends[b, at:at + n] = torch.arange(at + 1, at + n + 1, dtype=torch.int32)
            at += n
    return starts, ends


def _mask(gen, mask, B, S, S_kv):
    if mask == "docs":
        return dict(zip(("starts", "ends"), _docs(gen, B, S)))
    if mask == "window":  # a sliding window, some rows empty, some past both ends
        t = torch.arange(S).expand(B, S) + (S_kv - S)
        starts, ends = (t - 40).to(torch.int32), (t + 23).to(torch.int32)
        ends[:, ::5] = starts[:, ::5]
        return dict(starts=starts.contiguous(), ends=ends.contiguous())
    return dict(causal=mask == "causal")


def check(got, ref, names):
    for n in names:
        a, e, tol = got[n].detach().double().cpu(), ref[n], ref["e_" + n]
        assert a.shape == e.shape, n
        same = (a == e) | (a.isnan() & e.isnan())
        bad = ~((a - e).abs() <= tol) & ~same
        assert not bad.any(), (n, int(bad.sum()), a[bad][:4], e[bad][:4], tol[bad][:4])


def run_absorbed(dev, q, kv, d_v, do, scale, mask):
    q, kv = q.to(dev).requires_grad_(), kv.to(dev).requires_grad_()
    m = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in mask.items()}
    out, lse = ops.LatentMLA.apply(q, kv, scale, d_v, m.get("causal"), m.get("starts"), m.get("ends"))
    dq, dkv = torch.autograd.grad(out, (q, kv), do.to(dev))
    return dict(out=out, lse=lse, dq=dq, dkv=dkv)


def run_expanded(dev, q, k_nope, k_pe, v, do, scale, mask):
    leaves = [x.to(dev).requires_grad_() for x in (q, k_nope, k_pe, v)]
    m = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in mask.items()}
    out, lse = ops.LatentMLAExpanded.apply(*leaves, scale, m.get("causal"), m.get("starts"), m.get("ends"))
    grads = torch.autograd.grad(out, leaves, do.to(dev))
    return dict(zip(("out", "lse", "dq", "dk_nope", "dk_pe", "dv"), (out, lse, *grads)))


ABSORBED = [
    # B, S, S_kv, H, G, d_qk, d_v, mask
    (1, 1, 1, 1, 1, 128, 64, "causal"),
    (1, 1, 77, 16, 1, 128, 64, "causal"),
    (2, 5, 3, 4, 2, 128, 64, "causal"),        # the first queries precede every key
    (1, 64, 64, 32, 1, 128, 64, "causal"),
    (2, 129, 129, 28, 1, 128, 64, "causal"),
    (1, 200, 333, 8, 2, 128, 64, "full"),
    (2, 150, 150, 12, 1, 128, 64, "docs"),
    (1, 130, 190, 6, 3, 128, 64, "window"),
    (1, 700, 700, 2, 1, 128, 64, "causal"),
    (2, 96, 96, 5, 1, 128, 128, "causal"),
    (1, 131, 131, 3, 1, 128, 128, "docs"),
    (1, 100, 165, 16, 2, 192, 128, "causal"),
    (2, 77, 77, 7, 1, 192, 128, "window"),
]


@pytest.mark.parametrize("B,S,S_kv,H,G,d_qk,d_v,mask", ABSORBED)
def test_absorbed(dev, B, S, S_kv, H, G, d_qk, d_v, mask):
    gen = torch.Generator().manual_seed(S * 131 + H)
    q, kv, do = _normal(gen, B, S, H, d_qk), _normal(gen, B, S_kv, G, d_qk), _normal(gen, B, S, H, d_v)
    m = _mask(gen, mask, B, S, S_kv)
    ref = orc.absorbed(q, kv, d_v, d_qk ** -0.5, *orc.windows(B, S, S_kv, **m), do)
    check(run_absorbed(dev, q, kv, d_v, do, None, m), ref, ("out", "lse", "dq", "dkv"))


EXPANDED = [
    (1, 1, 1, 1, 192, 128, "causal"),
    (2, 3, 70, 4, 192, 128, "causal"),
    (1, 130, 130, 5, 192, 128, "causal"),
    (2, 90, 141, 3, 192, 128, "full"),
    (1, 260, 260, 2, 192, 128, "docs"),
    (1, 64, 128, 8, 128, 64, "causal"),
    (2, 133, 133, 6, 128, 64, "docs"),
    (1, 75, 140, 4, 128, 64, "window"),
    (1, 600, 600, 2, 128, 64, "causal"),
]


@pytest.mark.parametrize("B,S,S_kv,H,d_qk,d_v,mask", EXPANDED)
@pytest.mark.parametrize("views", [False, True])
def test_expanded(dev, B, S, S_kv, H, d_qk, d_v, mask, views):
    gen = torch.Generator().manual_seed(S * 17 + H)
    dn = d_qk - 64
    q, do = _normal(gen, B, S, H, d_qk), _normal(gen, B, S, H, d_v)
    up, pe = _normal(gen, B, S_kv, H, dn + d_v), _normal(gen, B, S_kv, 80)
    if views:  # one up-projection's rows, and the rope part of a down-projection's
        up, pe = up.to(dev), pe.to(dev)
    k_nope, v, k_pe = up[..., :dn], up[..., dn:], pe[..., 16:]
    if not views:
        k_nope, v, k_pe = k_nope.contiguous(), v.contiguous(), k_pe.contiguous()
    m = _mask(gen, mask, B, S, S_kv)
    ref = orc.expanded(q, k_nope.cpu(), k_pe.cpu(), v.cpu(), d_qk ** -0.5, *orc.windows(B, S, S_kv, **m), do)
    got = run_expanded(dev, q, k_nope, k_pe, v, do, None, m)
    check(got, ref, ("out", "lse", "dq", "dk_nope", "dk_pe", "dv"))
