"""Rotary positions fused with the q/k norms and the append to the pools (``tree_attention.rotary``).

Checked against the definition in 64 bits.  With y the normalised row, an output
a cos - b sin is rounded once to the type (``eps / 2`` relative to itself); the f32
steps before it (a mean of D squares, rsqrt, three products, sincospi at 2^-22
absolute, the fraction of a turn rounded to 2^-25 turns = 2^-22 rad) are within
``2^-20 (|a| + |b|) factor``.
"""
import math

import pytest
import torch

from tree_attention import _lib

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def inputs(n, hq, hk, dim, rot, dtype, seed, far=5000, norm=True):
    g = torch.Generator().manual_seed(seed)
    tokens = n + 17
    return dict(q=(torch.randn(n, hq, dim, generator=g) * 3).to(dtype).cuda(),
                k=(torch.randn(n, hk, dim, generator=g) * 3).to(dtype).cuda(),
                v=torch.randn(n, hk, dim, generator=g).to(dtype).cuda(),
                positions=torch.randint(0, far, (n,), generator=g).cuda(),
                inv_freq=(1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).float().cuda(),
                kp=torch.randn(hk, tokens, dim, generator=g).to(dtype).cuda(),
                vp=torch.randn(hk, tokens, dim, generator=g).to(dtype).cuda(),
                targets=torch.randperm(tokens, generator=g)[:n].cuda(),
                q_weight=(1 + torch.randn(dim, generator=g) / 4).to(dtype).cuda() if norm else None,
                k_weight=(1 + torch.randn(dim, generator=g) / 4).to(dtype).cuda() if norm else None)


def turned(x, weight, positions, inv_freq, interleaved=False, factor=1.0, eps=1e-6):
    """(rotated rows, sum of the magnitudes of a pair's terms), 64 bits."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    angle = (positions.double()[:, None] * inv_freq.double())[:, None]
    cos, sin = angle.cos() * factor, angle.sin() * factor
    rot = 2 * inv_freq.numel()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    ra, rb, size = a * cos - b * sin, b * cos + a * sin, (a.abs() + b.abs()) * factor
    pair = (lambda u, w: torch.stack((u, w), -1).flatten(-2)) if interleaved else (lambda u, w: torch.cat((u, w), -1))
    return torch.cat((pair(ra, rb), y[..., rot:]), -1), torch.cat((pair(size, size), y[..., rot:].abs()), -1)


def close(got, want, size):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    tol = half * want.abs() + 2.0 ** -20 * size + tiny
    off = (got.double() - want).abs()
    assert torch.all(off <= tol), f"worst {(off / tol).max():.3f} of the tolerance"


def run_and_check(x, interleaved=False, factor=1.0, **kwargs):
    from tree_attention.rotary import rotary_append
    kp, vp = x["kp"].clone(), x["vp"].clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = rotary_append(x["q"], x["k"], x["v"], x["positions"], x["inv_freq"], kp, vp, x["targets"],
                        interleaved=interleaved, attention_factor=factor, q_weight=x["q_weight"],
                        k_weight=x["k_weight"], status=status, **kwargs)
    torch.cuda.synchronize()
    assert int(status) == 0
    args = (x["positions"], x["inv_freq"], interleaved, factor)
    close(out, *turned(x["q"], x["q_weight"], *args))
    keep = x["targets"] >= 0
    where = x["targets"][keep]
    want, size = turned(x["k"], x["k_weight"], *args)
    close(kp[:, where].transpose(0, 1), want[keep], size[keep])
    assert torch.equal(vp[:, where].transpose(0, 1), x["v"][keep])
    rest = torch.ones(kp.shape[1], dtype=torch.bool, device="cuda")
    rest[where] = False
    assert torch.equal(kp[:, rest], x["kp"][:, rest]) and torch.equal(vp[:, rest], x["vp"][:, rest])
    return out


# ---- on the CPU ------------------------------------------------------------------
def test_validation_without_gpu():
    lib = _lib.load()
    p = 4096

    def call(q=p, st=4096, sh=128, k=p, v=p, pos=p, freq=p, rot=128, qw=p, out=p, kp=p, targets=p, n=2, hq=32, hk=8,
             tokens=64, dim=128, dtype=_lib.DTYPE_BF16, klen=None, tails=None, num_tails=0):
        return lib.ta_rotary_append(q, st, sh, k, 1024, 128, v, 1024, 128, pos, freq, rot, 0, 1.0, qw, None, 1e-6, out,
                                    kp, p, targets, n, hq, hk, tokens, dim, dtype, klen, tails, num_tails, None, 0, 4,
                                    None, None)

    assert call(dtype=_lib.DTYPE_F32) == _lib.ERR_UNSUPPORTED and call(dim=96) == _lib.ERR_UNSUPPORTED
    for bad in (dict(n=-1), dict(hq=-1), dict(tokens=-1), dict(rot=8), dict(rot=144), dict(rot=-16), dict(q=None),
                dict(q=p + 8), dict(st=4100), dict(sh=-128), dict(k=None), dict(v=p + 2), dict(pos=None),
                dict(freq=None), dict(out=None), dict(kp=None), dict(kp=p + 8), dict(targets=None), dict(qw=p + 2),
                dict(klen=p, num_tails=1)):
        assert call(**bad) == _lib.ERR_ARG, bad
    assert call(n=0) == 0                                    # nothing to do, nothing launched


def test_frequencies():
    from tree_attention.rotary import rotary_frequencies
    base, rot = 10000.0, 64
    i = torch.arange(0, rot, 2, dtype=torch.float64) / rot
    plain, factor = rotary_frequencies(rot, base)
    assert plain.dtype == torch.float32 and factor == 1.0 and torch.equal(plain, (base ** -i).float())
    assert torch.equal(rotary_frequencies(rot, base, dict(type="linear", factor=4.0))[0], (base ** -i / 4).float())
    # dynamic: nothing up to the trained length; beyond it the slowest pair turns 1 / stretch as fast
    dynamic = dict(type="dynamic", factor=2.0, original=4096)
    assert torch.equal(rotary_frequencies(rot, base, dynamic, length=100)[0], plain)
    longer = rotary_frequencies(rot, base, dynamic, length=16384)[0]
    assert longer[0] == 1 and math.isclose(longer[-1], plain[-1] / 7, rel_tol=1e-5)   # 2 * 4 - 1
    # yarn and bands: fast pairs keep their frequency, slow ones are divided, none leaves the range between
    for scaling, attention in ((dict(type="yarn", factor=8.0, original=4096), 0.1 * math.log(8.0) + 1),
                               (dict(type="bands", factor=8.0, original=8192, low=1.0, high=4.0), 1.0)):
        freq, factor = rotary_frequencies(rot, base, scaling)
        assert math.isclose(factor, attention)
        assert freq[0] == plain[0] and math.isclose(freq[-1], plain[-1] / 8, rel_tol=1e-6)
        assert torch.all(freq <= plain) and torch.all(freq >= plain / 8 * (1 - 1e-6))
    turns = 8192 * base ** -i / (2 * math.pi)
    freq = rotary_frequencies(rot, base, dict(type="bands", factor=8.0, original=8192, low=1.0, high=4.0))[0]
    assert torch.equal(freq[turns >= 4], plain[turns >= 4])
    assert torch.allclose(freq[turns <= 1], plain[turns <= 1] / 8)
    for bad in (dict(type="nope", factor=2.0), dict(factor=2.0), dict(type="linear", factor=0.5),
                dict(type="bands", factor=2.0, original=100, low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(rot, base, bad)
    for bad in ((0, 10.0), (3, 10.0), (4, 0.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(*bad)


# ---- on the GPU ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("shape", [(32, 8, 128, 128), (16, 2, 128, 96), (12, 4, 64, 64), (5, 5, 64, 16), (3, 1, 32, 32),
                                   (8, 8, 32, 16), (1, 1, 128, 0)], ids=lambda s: "x".join(map(str, s)))
def test_rotary_append(shape, interleaved, dtype):
    hq, hk, dim, rot = shape
    for n, norm in ((1, True), (19, False), (130, True)):
        x = inputs(n, hq, hk, dim, rot, DTYPES[dtype], n, norm=norm)
        run_and_check(x, interleaved, 1.0 if norm else 1.25)


@pytest.mark.gpu
def test_far_positions():
    """Angles of up to 10^9 rad, positions of every size."""
    x = inputs(40, 8, 2, 128, 128, torch.float16, 1)
    x["positions"] = torch.tensor([0, 1, 2 ** 20, 999_999_937] * 10).cuda()
    run_and_check(x)


@pytest.mark.gpu
def test_one_norm_only_and_extreme_rows():
    x = inputs(33, 8, 2, 128, 64, torch.bfloat16, 2)
    x["q_weight"] = None
    x["k"][3] = 0                                            # eps carries the norm of a zero row
    x["k"][4] *= 1e15
    run_and_check(x)


@pytest.mark.gpu
def test_slices_padding_and_in_place():
    """q, k and v as slices of one projection, padding targets, out = q, misaligned rows."""
    from tree_attention.rotary import rotary_append
    x = inputs(21, 8, 2, 64, 64, torch.bfloat16, 3)
    fused = torch.cat((x["q"], x["k"], x["v"]), 1)
    x["q"], x["k"], x["v"] = fused[:, :8], fused[:, 8:10], fused[:, 10:]
    x["targets"][5] = x["targets"][20] = -1
    want = run_and_check(x)
    odd = torch.zeros(21, 8, 65, device="cuda", dtype=torch.bfloat16)
    odd[..., 1:] = x["q"]
    x["q"] = odd[..., 1:]
    assert torch.equal(run_and_check(x), want)
    q = x["q"].contiguous()
    got = rotary_append(q, x["k"], x["v"], x["positions"], x["inv_freq"], x["kp"], x["vp"], x["targets"],
                        q_weight=x["q_weight"], k_weight=x["k_weight"], out=q)
    assert got is q and torch.equal(q, want)


@pytest.mark.gpu
def test_targets_outside_the_pools_are_recorded():
    from tree_attention.rotary import rotary_append
    x = inputs(6, 4, 2, 64, 64, torch.bfloat16, 4)
    before = x["kp"].clone(), x["vp"].clone()
    x["targets"] = torch.tensor([0, x["kp"].shape[1], -2, 3, 2 ** 40, -1]).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    rotary_append(x["q"], x["k"], x["v"], x["positions"], x["inv_freq"], x["kp"], x["vp"], x["targets"], status=status)
    assert int(status) == _lib.ERR_BOUNDS
    rest = [i for i in range(x["kp"].shape[1]) if i not in (0, 3)]
    assert torch.equal(x["kp"][:, rest], before[0][:, rest]) and torch.equal(x["vp"][:, rest], before[1][:, rest])
    assert torch.equal(x["vp"][:, [0, 3]].transpose(0, 1), x["v"][[0, 3]])


@pytest.mark.gpu
def test_refusals_on_gpu():
    from tree_attention.rotary import rotary_append
    x = inputs(4, 4, 2, 64, 64, torch.bfloat16, 5)
    rotary_append(**x)
    empty = {n: x[n][:0] for n in ("q", "k", "v", "positions", "targets")}
    assert rotary_append(**{**x, **empty}).shape == (0, 4, 64)
    for change in (dict(q=x["q"].float()), dict(q=x["q"][:3]), dict(k=x["k"][:, :1]), dict(v=x["v"].half()),
                   dict(positions=x["positions"].int()), dict(targets=x["targets"][:3]),
                   dict(positions=x["positions"].cpu()), dict(inv_freq=x["inv_freq"].double()),
                   dict(inv_freq=x["inv_freq"][:4]), dict(inv_freq=torch.ones(40, device="cuda")),
                   dict(kp=x["kp"].half()), dict(kp=x["kp"][:, ::2], vp=x["vp"][:, ::2]), dict(q_weight=torch.ones(64).cuda()),
                   dict(q_weight=x["q_weight"][:32]), dict(out=torch.empty(4, 4, 64)), dict(out=x["q"][:, :3]),
                   dict(out=x["kp"].flatten()[:4 * 4 * 64].view(4, 4, 64)), dict(status=torch.zeros(1).cuda())):
        with pytest.raises(ValueError):
            rotary_append(**{**x, **change})


@pytest.mark.gpu
def test_inputs_in_the_pools_are_refused():
    """Rows that lie in the pools would be read and written at once."""
    from tree_attention.rotary import rotary_append
    x = inputs(4, 4, 2, 64, 64, torch.bfloat16, 6)
    for change in (dict(k=x["kp"][:, 3:7].transpose(0, 1)), dict(v=x["vp"][:, 3:7].transpose(0, 1)),
                   dict(q=x["vp"].flatten()[64:64 + 4 * 4 * 64].view(4, 4, 64))):
        with pytest.raises(ValueError):
            rotary_append(**{**x, **change})
