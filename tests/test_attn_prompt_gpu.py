"""GPU: causal attention over packed prompts against a 64-bit restatement.  Tolerances come from the roundings of each type
(serving_util.prompt_tolerance) and, for f32, a bound of 1e-5 on the relative 2-norm of the error."""
import math

import pytest
import torch

from serving_util import TYPES, attend64, back, code, dev, half_ulp, i32, offsets, prompt_tolerance

pytestmark = pytest.mark.gpu


def inputs(seed, dtype, H, G, D, nq, before, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    nk = [max(0, a + b) for a, b in zip(nq, before)]
    r = lambda n, h, s=1.0: (torch.randn(n, h, D, generator=g) * s).to(TYPES[dtype])
    return r(sum(nq), H, gain), r(sum(nk), G), r(sum(nk), G), nq, nk


def run(gpu, dtype, q, k, v, nq, nk, scale, tail=0, same=False, out=None):
    H, D, G = q.shape[1], q.shape[2], k.shape[1]
    out = torch.full((q.shape[0] + tail, H, D), 7.0, dtype=TYPES[dtype]) if out is None else out
    qq = torch.cat([q, torch.full((tail, H, D), math.nan, dtype=q.dtype)])
    bufs = [dev(gpu, t) for t in (qq, k, v, out, offsets(nq), offsets(nk))]
    gpu.attn_prompt(bufs[0], bufs[1], bufs[2], bufs[3], bufs[4], None if same else bufs[5], len(nq), qq.shape[0],
                    qq.shape[0] if same else k.shape[0], H, G, D, scale=scale, dtype=code(gpu, dtype))
    got = back(gpu, bufs[3], out)
    gpu.check(gpu.lib().simp_gpu_check_device_status())
    return got


def reference(q, k, v, nq, nk, scale):
    out, a, b = [], 0, 0
    for n, m in zip(nq, nk):
        out.append(attend64(q[a:a + n], k[b:b + m], v[b:b + m], scale))
        a, b = a + n, b + m
    return torch.cat(out)


def compare(got, ref, q, k, v, nk, scale, dtype, norm=True):
    t = TYPES[dtype]
    fine = torch.isfinite(ref)
    assert torch.equal(fine, torch.isfinite(got.double()))
    tol = prompt_tolerance(q, k, v, scale, max(nk), t, dtype != "f32") + half_ulp(t) * ref.abs()
    err = (got.double() - ref).abs()
    assert bool((err[fine] <= tol[fine] + 1e-30).all()), f"largest error {err[fine].max()} at tolerance {tol[fine].min()}"
    if norm and dtype == "f32" and ref[fine].norm() > 0:
        assert err[fine].norm() <= 1e-5 * ref[fine].norm()


SHAPES = [
    # heads, kv heads, head_dim, queries per sequence, cached keys before them
    (1, 1, 64, [1], [0]),
    (2, 1, 128, [2, 1, 0, 3], [0, 5, 0, 0]),
    (4, 4, 64, [63, 64, 65], [0, 0, 0]),
    (8, 2, 128, [127, 128, 129, 1], [0, 1, 0, 200]),
    (12, 12, 64, [257, 31], [0, 0]),
    (32, 8, 64, [96, 0, 0, 33, 300], [0, 0, 7, 0, 150]),
    (6, 2, 128, [150, 43], [0, 90]),          # groups of three heads: tiles of 42 tokens
    (5, 1, 64, [70, 200], [0, 11]),
    (16, 1, 128, [40, 9], [0, 300]),
    (40, 8, 128, [77], [0]),
    (8, 1, 64, [513], [0]),
    (2, 2, 128, [640], [0]),
    (32, 32, 100, [70, 5], [0, 20]),          # head sizes that are no power of two
    (3, 3, 16, [50, 1], [0, 2]),
    (4, 2, 33, [20, 130], [0, 0]),
    (2, 1, 1, [9], [0]),
    (4, 4, 96, [140], [0]),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "h%dg%dd%d_%s" % (s[0], s[1], s[2], "-".join(map(str, s[3]))))
def test_against_64_bits(gpu, dtype, shape):
    H, G, D, nq, before = shape
    q, k, v, nq, nk = inputs(H * 1000 + D, dtype, H, G, D, nq, before)
    scale = D ** -0.5
    got = run(gpu, dtype, q, k, v, nq, nk, scale)
    compare(got, reference(q, k, v, nq, nk, scale), q, k, v, nk, scale, dtype)


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("bf16", 128), ("f16", 64)])
def test_one_long_sequence(gpu, dtype, D):
    q, k, v, nq, nk = inputs(5, dtype, 2, 1, D, [2500], [0])
    got = run(gpu, dtype, q, k, v, nq, nk, D ** -0.5, same=True)
    compare(got, reference(q, k, v, nq, nk, D ** -0.5), q, k, v, nk, D ** -0.5, dtype)


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("bf16", 128), ("f16", 64), ("bf16", 40)])
def test_many_sequences_and_rows_behind_the_last(gpu, dtype, D):
    """More sequences than are looked at together, and rows that belong to none: left as they were."""
    nq = [(i * 7) % 23 for i in range(70)]
    q, k, v, nq, nk = inputs(6, dtype, 4, 2, D, nq, [0] * 70)
    got = run(gpu, dtype, q, k, v, nq, nk, 0.2, tail=37)
    assert bool((got[sum(nq):] == 7.0).all())
    compare(got[:sum(nq)], reference(q, k, v, nq, nk, 0.2), q, k, v, nk, 0.2, dtype)


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("bf16", 128), ("f16", 64), ("f16", 128)])
def test_rows_that_see_nothing(gpu, dtype, D):
    """More queries than keys: the first rows see nothing and get zeros, also where a whole tile sees nothing."""
    nq, nk = [300, 5, 140], [20, 0, 139]
    q, _, _, _, _ = inputs(7, dtype, 4, 4, D, nq, [0, 0, 0])
    _, k, v, _, _ = inputs(8, dtype, 4, 4, D, nk, [0, 0, 0])
    got = run(gpu, dtype, q, k, v, nq, nk, D ** -0.5)
    ref = reference(q, k, v, nq, nk, D ** -0.5)
    assert bool((got[:280] == 0).all()) and bool((got[300:305] == 0).all()) and bool((got[305] == 0).all())
    compare(got, ref, q, k, v, nk, D ** -0.5, dtype)


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("bf16", 128), ("f16", 64), ("bf16", 64), ("f32", 100)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_has_no_influence(gpu, dtype, D, bad):
    """NaN or infinity in keys and values: rows before them and other sequences are exactly as without them, rows after them
    show them as the formula does."""
    q, k, v, nq, nk = inputs(9, dtype, 4, 2, D, [150, 37, 290], [0, 0, 0])
    clean = run(gpu, dtype, q, k, v, nq, nk, D ** -0.5)
    place = 187 + 200            # row 200 of the last sequence
    v2 = v.clone()
    v2[place, 1, 3] = bad
    got = run(gpu, dtype, q, k, v2, nq, nk, D ** -0.5)
    assert torch.equal(got[:place], clean[:place])
    seen = got[place:, 2:, 3].double()
    assert bool((torch.isnan(seen) if math.isnan(bad) else seen == bad).all())
    rest = torch.ones(got.shape[1:], dtype=torch.bool)
    rest[2:, 3] = False
    assert torch.equal(got[place:][:, rest], clean[place:][:, rest])
    k2 = k.clone()
    k2[place, 1, :] = bad
    got = run(gpu, dtype, q, k2, v, nq, nk, D ** -0.5)
    assert torch.equal(got[:place], clean[:place]) and torch.equal(got[:, :2], clean[:, :2])


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("bf16", 128), ("f16", 64)])
def test_large_scores(gpu, dtype, D):
    """Scores of several hundred: the running maximum has to move, and weights underflow instead of overflowing."""
    q, k, v, nq, nk = inputs(10, dtype, 2, 1, D, [400], [0], gain=30.0)
    k[0::3] *= 4
    got = run(gpu, dtype, q, k, v, nq, nk, 1.0)
    # scores of 1000 are off by 2^-24 of that per operation, and weights by as much relative: no bound on the 2-norm here
    compare(got, reference(q, k, v, nq, nk, 1.0), q, k, v, nk, 1.0, dtype, norm=False)


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_any_scale(gpu, dtype, D, scale):
    q, k, v, nq, nk = inputs(11, dtype, 2, 2, D, [200], [0])
    got = run(gpu, dtype, q, k, v, nq, nk, scale)
    compare(got, reference(q, k, v, nq, nk, scale), q, k, v, nk, abs(scale), dtype)


@pytest.mark.parametrize("dtype,D,pad,first", [("bf16", 128, 0, 0), ("bf16", 128, 8, 8), ("f16", 64, 24, 0), ("f16", 64, 3, 1), ("f32", 64, 5, 3), ("bf16", 64, 4, 0)])
def test_parts_of_one_projection(gpu, dtype, D, pad, first):
    """q, k and v side by side in one tensor, rows a stride apart that need not be a multiple of 16 bytes, output too."""
    H, G, nq = 8, 2, [130, 77]
    t, n, es = TYPES[dtype], 207, TYPES[dtype].itemsize
    width = (H + 2 * G) * D + pad
    g = torch.Generator().manual_seed(12)
    x = torch.randn(n * width + first, generator=g).to(t)
    rows = x[first:].view(n, width)
    q, k, v = rows[:, :H * D].reshape(n, H, D), rows[:, H * D:(H + G) * D].reshape(n, G, D), rows[:, (H + G) * D:(H + 2 * G) * D].reshape(n, G, D)
    ow = H * D + pad
    out = torch.full((n, ow), 7.0, dtype=t)
    bx, bo, off = dev(gpu, x), dev(gpu, out), dev(gpu, offsets(nq))
    at = lambda i: bx.offset((first + i) * es)
    gpu.attn_prompt(at(0), at(H * D), at((H + G) * D), bo, off, None, 2, n, n, H, G, D, q_stride=width, kv_stride=width, out_stride=ow, dtype=code(gpu, dtype))
    got = back(gpu, bo, out)
    assert bool((got[:, H * D:] == 7.0).all())
    scale = D ** -0.5
    compare(got[:, :H * D].reshape(n, H, D), reference(q, k, v, nq, nq, scale), q, k, v, nq, scale, dtype)


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("bf16", 128)])
def test_bad_offsets_are_reported_and_skipped(gpu, dtype, D):
    t = TYPES[dtype]
    x = torch.randn(60, 2, D).to(t)
    for off in ([0, 30, 20, 60], [0, 10, 20, 61], [-1, 5, 9, 60], [0, 2 ** 31 - 1, 3, 60]):
        out = torch.full((60, 2, D), 7.0, dtype=t)
        b, bo, bf = dev(gpu, x), dev(gpu, out), dev(gpu, i32(off))
        gpu.attn_prompt(b, b, b, bo, bf, None, 3, 60, 60, 2, 2, D, dtype=code(gpu, dtype))
        with pytest.raises(gpu.SimpGpuError, match="out of range"):
            gpu.check(gpu.lib().simp_gpu_check_device_status())
        assert bool(torch.isfinite(back(gpu, bo, out).float()).all())
    gpu.check(gpu.lib().simp_gpu_check_device_status())   # reported once, usable again
    got = run(gpu, dtype, x, x, x, [60], [60], 0.1)
    compare(got, reference(x, x, x, [60], [60], 0.1), x, x, x, [60], 0.1, dtype)


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("bf16", 128), ("f16", 64)])
def test_recorded_and_repeated(gpu, dtype, D):
    """The same call gives the same bits each time, recorded too, with other inputs in the same buffers."""
    q, k, v, nq, nk = inputs(13, dtype, 8, 2, D, [200, 90], [0, 0])
    out = torch.zeros_like(q)
    b = [dev(gpu, t) for t in (q, k, v, out, offsets(nq))]
    call = lambda: gpu.attn_prompt(b[0], b[1], b[2], b[3], b[4], None, 2, 290, 290, 8, 2, D, dtype=code(gpu, dtype))
    call()
    first = back(gpu, b[3], out)
    with gpu.Recording() as rec:
        call()
    b[3].zero()
    rec.replay(2)
    assert torch.equal(back(gpu, b[3], out), first)
    b[0].upload(dev_bytes(-q))
    rec.replay(1)
    got = back(gpu, b[3], out)
    rec.close()
    assert torch.equal(got, run(gpu, dtype, -q, k, v, nq, nk, D ** -0.5)) and not torch.equal(got, first)


def dev_bytes(t):
    return t.contiguous().view(torch.uint8).numpy().reshape(-1)
