"""The oracles of layer norm and of the index keys against differences, torch's own layer norm and exhaustive codes."""
import math

import pytest
import torch

from oracle import index_keys as ok
from oracle import layer_norm as ol


@pytest.mark.parametrize("affine", [True, False])
def test_layer_norm_gradients(affine):
    gen = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(5, 11, generator=gen, dtype=torch.float64) for _ in range(2))
    w, b = (torch.randn(11, generator=gen, dtype=torch.float64) for _ in range(2)) if affine else (None, None)
    r = ol.layer_norm(x, w, b, 1e-5, dy)
    assert torch.allclose(r["y"], torch.nn.functional.layer_norm(x, (11,), w, b, 1e-5), atol=1e-12)
    f = lambda x, w, b: float((ol.layer_norm(x, w, b, 1e-5)["y"] * dy).sum())  # noqa: E731
    h = 1e-6
    for name, at in (("dx", 0), ("dweight", 1), ("dbias", 2)):
        args = [x, w, b]
        if args[at] is None:
            continue
        flat = r[name].flatten()
        for i in range(flat.numel()):
            step = torch.zeros_like(args[at]).flatten()
            step[i] = h
            up, down = list(args), list(args)
            up[at], down[at] = args[at] + step.view_as(args[at]), args[at] - step.view_as(args[at])
            assert abs((f(*up) - f(*down)) / (2 * h) - float(flat[i])) < 1e-7, (name, i)


def test_e4m3_values():
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(codes, torch.tensor(ok.E4M3, dtype=torch.float64))
    x = torch.cat([torch.rand(200, dtype=torch.float64) * s for s in (0.01, 1, 30, 448)]).float()
    assert [ok._nearest_e4m3(float(v)) for v in x] == x.to(torch.float8_e4m3fn).view(torch.uint8).tolist()


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("d", [64, 128])
def test_pack_and_unpack(fmt, d):
    gen = torch.Generator().manual_seed(d)
    k = (torch.randn(16, d, generator=gen) * torch.exp2(torch.randint(-20, 20, (16, 1), generator=gen).float())).to(torch.bfloat16)
    packed = [ok.pack_key(x, fmt) for x in k]
    page = torch.tensor(sum((c for c, _ in packed), []) + sum((e for _, e in packed), []), dtype=torch.uint8)
    back = ok.unpack_pages(page.view(1, 16, -1), d)
    x = k.double().unflatten(1, (-1, 32))
    step = 2.0 ** -4 if fmt == "mxfp8" else 2.0 ** -2                      # half a step; saturation of 6 .. 8: a quarter of 8
    least = x.abs().amax(-1, keepdim=True) * (2.0 ** -10 / 224 if fmt == "mxfp8" else 0.25 / 4)   # of what is subnormal
    assert ((back.unflatten(1, (-1, 32)) - x).abs() <= torch.maximum(step * x.abs(), least)).all()


def test_scores_of_one_key():
    q, k = torch.ones(1, 16, 64, dtype=torch.bfloat16), torch.full((4, 64), 0.5, dtype=torch.float64)
    w = torch.arange(16.0)[None]
    s, tol, n = ok.scores(q, w, k, torch.zeros(1, 1, dtype=torch.int32), [0, 1], [3], 4, 4)
    assert s[0].tolist() == [3840.0] * 3 + [-math.inf] and n.tolist() == [3]
    assert (ok.scores(-q, w, k, torch.zeros(1, 1, dtype=torch.int32), [0, 1], [3], 4, 4)[0][0, :3] == 0).all()
