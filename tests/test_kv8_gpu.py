"""GPU: the 8-bit key/value cache.  Writing is exact (integers and scales equal the 64-bit restatement's), reading back is
one rounding, attention is held to tolerances from the roundings of queries, weights and sums."""
import math

import numpy as np
import pytest
import torch

from serving_util import TYPES, Cache64, DeviceCache, attend64, back, code, dev, half_ulp, i32, make_table, offsets

pytestmark = pytest.mark.gpu


def rows(rng, n, heads, dim, dtype, gain=1.0):
    x = torch.from_numpy(rng.standard_normal((n, heads, dim)) * gain).to(TYPES[dtype])
    return x


def append(gpu, dc, table, k, v, lengths, starts, dtype, **more):
    bt = dev(gpu, torch.from_numpy(table))
    bufs = [dev(gpu, t) for t in (k, v, offsets(lengths), i32(starts))]
    gpu.kv8_append(dc.handle, bt, table.shape[1], *bufs, len(lengths), k.shape[0], dtype=code(gpu, dtype), **more)
    gpu.sync()


def same(dc, c64):
    q, s = dc.contents()
    for w in range(2):
        assert np.array_equal(s[w].view(np.uint32), c64.s[w].view(np.uint32)), "scales differ"
        assert np.array_equal(q[w], c64.q[w]), f"{(q[w] != c64.q[w]).sum()} integers differ"


def split(x, lengths):
    return list(torch.split(x, lengths))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bt,heads,dim,lengths", [(16, 1, 64, [1]), (16, 2, 128, [16, 17, 0, 15]), (32, 3, 100, [64, 1, 33]), (64, 8, 64, [200, 63]),
                                                  (128, 2, 16, [129, 128, 5]), (64, 1, 1, [70]), (32, 2, 33, [40, 90]), (64, 2, 96, [65])])
def test_append_to_empty_blocks(gpu, dtype, bt, heads, dim, lengths):
    rng = np.random.default_rng(bt + dim)
    table, blocks = make_table(lengths, bt, rng, extra=2)
    c64 = Cache64(blocks, bt, heads, dim, rng)
    dc = DeviceCache(gpu, c64)
    k, v = rows(rng, sum(lengths), heads, dim, dtype), rows(rng, sum(lengths), heads, dim, dtype, 0.01)
    append(gpu, dc, table, k, v, lengths, [0] * len(lengths), dtype)
    c64.append(table, list(zip(split(k.double(), lengths), split(v.double(), lengths))), [0] * len(lengths))
    same(dc, c64)
    gpu.check(gpu.lib().simp_gpu_check_device_status())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bt,dim", [(16, 64), (32, 100), (64, 128), (128, 40)])
def test_append_in_pieces(gpu, dtype, bt, dim):
    """Pieces of any length, values that grow and shrink: blocks are re-scaled as they fill, token by token and in runs."""
    rng = np.random.default_rng(dim)
    heads, total = 3, [3 * bt + 5, 2 * bt, bt // 2, 40]
    table, blocks = make_table(total, bt, rng, extra=1)
    c64 = Cache64(blocks, bt, heads, dim, rng)
    dc = DeviceCache(gpu, c64)
    at = [0] * len(total)
    for step in range(60):
        n = [min(t - a, int(rng.integers(0, 3 if step % 4 else bt))) for t, a in zip(total, at)]
        gain = 2.0 ** rng.integers(-3, 4)
        k, v = rows(rng, sum(n), heads, dim, dtype, gain), rows(rng, sum(n), heads, dim, dtype, 1 / gain)
        append(gpu, dc, table, k, v, n, at, dtype)
        c64.append(table, list(zip(split(k.double(), n), split(v.double(), n))), at)
        at = [a + b for a, b in zip(at, n)]
        if step % 10 == 0 or at == total:
            same(dc, c64)
        if at == total:
            break
    assert at == total


def test_values_next_to_halves(gpu):
    """Quotients that are halves, or as near to one as the type allows: to even, and to the side on which they lie."""
    bt, dim = 64, 64
    rng = np.random.default_rng(0)
    c64 = Cache64(64, bt, 1, dim)
    dc = DeviceCache(gpu, c64)
    table = np.arange(64, dtype=np.int32)[None]
    x = np.zeros((64, bt, dim), np.float32)
    for b in range(64):
        top = np.float32(127.0 if b == 0 else 2.0 ** rng.uniform(-60, 60))
        s = np.float32(top / np.float32(127))
        half = ((rng.integers(-127, 127, (bt, dim)) + 0.5) * float(s)).astype(np.float32)
        x[b] = np.nextafter(half, np.where(rng.random(half.shape) < 0.3, half, np.where(rng.random(half.shape) < 0.5, np.inf, -np.inf)).astype(np.float32))
        x[b] = np.clip(x[b], -top, top)
        x[b, 0, 0] = top
    k = torch.from_numpy(x.reshape(-1, 1, dim))
    append(gpu, dc, table, k, -k, [64 * bt], [0], "f32")
    c64.append(table, [(k.double(), -k.double())], [0])
    same(dc, c64)


def test_zeros_tiny_and_not_finite(gpu):
    bt, dim = 16, 32
    c64 = Cache64(6, bt, 1, dim)
    dc = DeviceCache(gpu, c64)
    table = np.arange(6, dtype=np.int32)[None]
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, bt, dim)).astype(np.float32)
    x[0] = 0
    x[1] *= 1e-38                       # scale below FLT_MIN: held as zeros
    x[2, 3, 4:9] = [np.nan, np.inf, -np.inf, 3.0e38, -3.0e38]
    x[3, :, :] = np.nan
    x[4, 0, 0] = np.inf
    x[5] *= 1e38
    x[5] = np.clip(x[5], -3.4e38, 3.4e38)
    k = torch.from_numpy(x.reshape(-1, 1, dim))
    append(gpu, dc, table, k, k, [6 * bt], [0], "f32")
    c64.append(table, [(k.double(), k.double())], [0])
    same(dc, c64)
    # into blocks that hold zeros only
    append(gpu, dc, np.array([[0]], np.int32), k[:4] + 1, k[:4], [4], [8], "f32")
    c64.append(np.array([[0]]), [(k[:4].double() + 1, k[:4].double())], [8])
    same(dc, c64)


@pytest.mark.parametrize("dtype,pad,first", [("f32", 3, 1), ("bf16", 1, 1), ("f16", 16, 8)])
def test_strided_rows(gpu, dtype, pad, first):
    """k and v as parts of one projection's rows, and rows behind the last sequence (garbage) left out."""
    rng = np.random.default_rng(2)
    heads, dim, bt, lengths = 2, 64, 32, [45, 30]
    t, es = TYPES[dtype], TYPES[dtype].itemsize
    width = 2 * heads * dim + pad
    x = torch.from_numpy(rng.standard_normal(80 * width + first)).to(t)
    r = x[first:].view(80, width)
    k, v = r[:75, :heads * dim].reshape(75, heads, dim), r[:75, heads * dim:2 * heads * dim].reshape(75, heads, dim)
    r[75:] = math.nan
    table, blocks = make_table(lengths, bt, rng)
    c64 = Cache64(blocks, bt, heads, dim)
    dc = DeviceCache(gpu, c64)
    bx, tb, off, st = dev(gpu, x), dev(gpu, torch.from_numpy(table)), dev(gpu, offsets(lengths)), dev(gpu, i32([0, 0]))
    gpu.kv8_append(dc.handle, tb, table.shape[1], bx.offset(first * es), bx.offset((first + heads * dim) * es), off, st, 2, 80, kv_stride=width, dtype=code(gpu, dtype))
    gpu.sync()
    c64.append(table, list(zip(split(k.double(), lengths), split(v.double(), lengths))), [0, 0])
    same(dc, c64)
    # and back into such rows
    out = torch.full((80, width), 5.0, dtype=t)
    bo = dev(gpu, out)
    gpu.kv8_read(dc.handle, tb, table.shape[1], bo.ptr, bo.offset(heads * dim * es), off, st, 2, 80, kv_stride=width, dtype=code(gpu, dtype))
    got = back(gpu, bo, out)
    assert bool((got[75:] == 5.0).all()) and bool((got[:, 2 * heads * dim:] == 5.0).all())
    for w in range(2):
        want = np.concatenate([c64.values(table[s], n, w) for s, n in enumerate(lengths)])
        part = got[:75, w * heads * dim:(w + 1) * heads * dim].reshape(75, heads, dim).double().numpy()
        assert np.all(np.abs(part - want) <= (half_ulp(t) + 2.0 ** -24) * np.abs(want) * 1.0001)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bt,dim", [(16, 64), (32, 100), (64, 128), (128, 17)])
def test_read(gpu, dtype, bt, dim):
    """integer * scale is one f32 rounding (2^-24), then one to the type."""
    rng = np.random.default_rng(3)
    lengths = [150, 1, 0, 77]
    table, blocks = make_table(lengths, bt, rng)
    c64 = Cache64(blocks, bt, 2, dim, rng)
    dc = DeviceCache(gpu, c64)
    starts, n = [20, 0, 0, 76], [130, 1, 0, 1]
    t = TYPES[dtype]
    out = torch.zeros(sum(n), 2, dim, dtype=t)
    bk, bv = dev(gpu, out), dev(gpu, out)
    gpu.kv8_read(dc.handle, dev(gpu, torch.from_numpy(table)), table.shape[1], bk, bv, dev(gpu, offsets(n)), dev(gpu, i32(starts)), 4, sum(n), dtype=code(gpu, dtype))
    for w, b in enumerate((bk, bv)):
        want = np.concatenate([c64.values(table[s], starts[s] + n[s], w)[starts[s]:] for s in range(4)])
        got = back(gpu, b, out).double().numpy()
        assert np.all(np.abs(got - want) <= (half_ulp(t) + 2.0 ** -24) * np.abs(want) * 1.0001)


def test_bad_blocks_and_places_are_reported_and_skipped(gpu):
    rng = np.random.default_rng(4)
    bt, dim = 16, 64
    c64 = Cache64(4, bt, 2, dim, rng)
    dc = DeviceCache(gpu, c64)
    k = rows(rng, 40, 2, dim, "f32")
    status = lambda: gpu.check(gpu.lib().simp_gpu_check_device_status())
    for table, lengths, starts in (([[0, 4]], [20], [0]), ([[-1, 1]], [20], [0]), ([[0, 2 ** 31 - 1]], [20], [0]), ([[0, 1]], [33], [0]), ([[0, 1]], [20], [13]),
                                   ([[0, 1]], [20], [-1])):
        append(gpu, dc, np.array(table, np.int32), k, k, lengths, starts, "f32")
        with pytest.raises(gpu.SimpGpuError, match="outside the cache|out of range"):
            status()
    q, s = dc.contents()
    assert all(np.array_equal(q[w][2:], c64.q[w][2:]) and np.array_equal(s[w][2:], c64.s[w][2:]) for w in range(2))
    status()
    # attention: a block outside the cache has no weight, the others count
    table = np.array([[2, 9, 3]], np.int32)
    c64.q, c64.s = [a.copy() for a in q], [a.copy() for a in s]
    qq = rows(rng, 1, 2, dim, "f32")
    out = torch.zeros(1, 2, dim)
    bo = dev(gpu, out)
    gpu.attn_kv8(dc.handle, dev(gpu, torch.from_numpy(table)), 3, dev(gpu, qq), bo, dev(gpu, i32([44])), 1, 48, 2)
    with pytest.raises(gpu.SimpGpuError, match="outside the cache"):
        status()
    kk, vv = ([c64.values([2], 16, w), c64.values([3], 12, w)] for w in range(2))
    ref = attend64(qq, torch.from_numpy(np.concatenate(kk)), torch.from_numpy(np.concatenate(vv)), dim ** -0.5)
    assert float((back(gpu, bo, out).double() - ref).abs().max()) < 1e-5
    # lengths that the call did not announce: reported, the output left as it was
    for n in (49, -1):
        bo = dev(gpu, out + 7)
        gpu.attn_kv8(dc.handle, dev(gpu, torch.from_numpy(table)), 3, dev(gpu, qq), bo, dev(gpu, i32([n])), 1, 48, 2)
        with pytest.raises(gpu.SimpGpuError, match="out of range"):
            status()
        assert bool((back(gpu, bo, out) == 7).all())


# ------------------------------------------------------------------------------------------------ attention
def attention_tolerance(c64, table, lengths, q, scale, dtype, ref):
    """Queries become integers relative to their largest element (half a step of 1 / 32512, f32: of 2^-22.99), so a score is off by
    that times scale sum_d |k_d|, plus f32 roundings of the score itself; weights carry it twice (numerator, denominator) and
    2^-20 of exponentials; as integers they are off by half of 1 / 65535 (f32: 2^-24) of the largest of their 32, which is at
    most 32 / 65535 / 2 of the whole; sums of n / 32 tile results are f32.  One output rounding."""
    t = TYPES[dtype]
    step, weight = (0.5 / (127 << 16), 32 * 0.5 / 16777215) if dtype == "f32" else (0.5 / 32512, 32 * 0.5 / 65535)
    tol = 0.0
    for s, n in enumerate(lengths):
        if not n:
            continue
        used = table[s][:(n + c64.bt - 1) // c64.bt]
        kmax = 127 * c64.s[0][used].max()
        vmax = 127 * c64.s[1][used].max()
        qmax = float(q[s].double().abs().max())
        ds = abs(scale) * qmax * kmax * c64.dim * (step + 2.0 ** -21)
        tol = max(tol, float(vmax * (2 * ds + 2.0 ** -20 + weight + (n / 32 + 20) * 2.0 ** -23)))
    return tol + half_ulp(t) * ref.abs()


def attention(gpu, dc, table, q, lengths, scale, dtype, max_len=None):
    out = torch.full(q.shape, 7.0, dtype=q.dtype)
    bo = dev(gpu, out)
    gpu.attn_kv8(dc.handle, dev(gpu, torch.from_numpy(table)), table.shape[1], dev(gpu, q), bo, dev(gpu, i32(lengths)), len(lengths),
                 max(lengths) if max_len is None else max_len, q.shape[1], scale=scale, dtype=code(gpu, dtype))
    got = back(gpu, bo, out)
    gpu.check(gpu.lib().simp_gpu_check_device_status())
    return got


def reference(c64, table, q, lengths, scale):
    out = []
    for s, n in enumerate(lengths):
        k, v = (torch.from_numpy(c64.values(table[s], n, w)) for w in range(2))
        out.append(attend64(q[s:s + 1], k, v, scale))
    return torch.cat(out)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,dim,bt,lengths", [
    (1, 1, 64, 16, [1]), (2, 1, 128, 16, [15, 16, 17, 0]), (4, 1, 64, 32, [31, 32, 33, 129]), (8, 2, 128, 64, [500, 1, 63, 64, 65]),
    (8, 1, 64, 64, [700, 20]), (5, 1, 100, 16, [130, 7]), (12, 1, 128, 32, [300]), (32, 2, 64, 128, [260, 128]), (6, 2, 32, 16, [90, 40]),
    (3, 3, 16, 32, [70]), (7, 1, 96, 64, [222, 3]), (32, 32, 100, 16, [60, 0, 3]), (16, 1, 1, 16, [50]), (9, 3, 40, 128, [300, 2])])
def test_attention_against_64_bits(gpu, dtype, H, G, dim, bt, lengths):
    rng = np.random.default_rng(H * 100 + dim)
    table, blocks = make_table(lengths, bt, rng, extra=1)
    c64 = Cache64(blocks, bt, G, dim, rng)
    dc = DeviceCache(gpu, c64)
    q = rows(rng, len(lengths), H, dim, dtype)
    scale = dim ** -0.5
    got, ref = attention(gpu, dc, table, q, lengths, scale, dtype), reference(c64, table, q, lengths, scale)
    err = (got.double() - ref).abs()
    assert bool((err <= attention_tolerance(c64, table, lengths, q, scale, dtype, ref)).all()), float(err.max())
    if dtype == "f32":
        assert err.norm() <= 1e-5 * ref.norm()


@pytest.mark.parametrize("dtype,H,G,dim", [("f32", 4, 1, 64), ("bf16", 8, 1, 128), ("f16", 8, 2, 64)])
def test_long_cache_is_split_and_joined(gpu, dtype, H, G, dim):
    """Several thousand tokens over many blocks of the GPU, beside sequences that need one; scales that differ a lot from
    block to block; the same bits each time, recorded too."""
    rng = np.random.default_rng(5)
    lengths, bt = [6007, 10, 0, 2500], 32
    table, blocks = make_table(lengths, bt, rng)
    c64 = Cache64(blocks, bt, G, dim, rng)
    for w in range(2):
        c64.s[w] *= (2.0 ** rng.integers(-4, 3, c64.s[w].shape)).astype(np.float32)
    dc = DeviceCache(gpu, c64)
    q = rows(rng, len(lengths), H, dim, dtype)
    scale = dim ** -0.5
    got, ref = attention(gpu, dc, table, q, lengths, scale, dtype), reference(c64, table, q, lengths, scale)
    err = (got.double() - ref).abs()
    assert bool((err <= attention_tolerance(c64, table, lengths, q, scale, dtype, ref)).all()), float(err.max())
    assert torch.equal(got, attention(gpu, dc, table, q, lengths, scale, dtype))
    out = torch.zeros_like(got)
    b = [dev(gpu, t) for t in (torch.from_numpy(table), q, out, i32(lengths))]
    with gpu.Recording() as rec:
        gpu.attn_kv8(dc.handle, b[0], table.shape[1], b[1], b[2], b[3], 4, 6007, H, dtype=code(gpu, dtype))
    with gpu.Recording() as rec2:     # a second recording on the same scratch
        gpu.attn_kv8(dc.handle, b[0], table.shape[1], b[1], b[2], b[3], 4, 6007, H, scale=0.0, dtype=code(gpu, dtype))
    rec2.replay(1)
    rec.replay(2)
    assert torch.equal(back(gpu, b[2], out), got)
    b[3].upload(np.array([100, 9, 0, 1500], np.int32))            # lengths are read on the device, at each replay
    rec.replay(1)
    assert torch.equal(back(gpu, b[2], out), attention(gpu, dc, table, q, [100, 9, 0, 1500], scale, dtype, max_len=6007))
    rec.close()
    rec2.close()


@pytest.mark.parametrize("factor", [2, 3, 6, 10, 1.5, 1.0078125, 63.5, 254])
@pytest.mark.parametrize("step", [1.0, 0.3, 3e-38])
def test_larger_steps_keep_halves_even(gpu, factor, step):
    """A block that grows by a factor that puts many held integers on halves: q old / new rounded to even, exactly."""
    bt, dim, held = 64, 32, 45
    step = np.float32(step)
    q = ((np.arange(held * dim) * 37) % 255 - 127).reshape(held, 1, dim)
    q[0, 0, 0] = 127
    first = (q * step).astype(np.float32)
    old = np.float32(np.abs(first).max() / np.float32(127.0))
    assert np.array_equal(np.rint(first.astype(np.float64) / old), q)
    last = np.zeros((1, 1, dim), np.float32)
    last[0, 0, 5] = -np.float32(127.0) * np.float32(factor) * step
    new = np.float32(np.abs(last).max() / np.float32(127.0))
    want = np.rint(q.astype(np.float64) * np.float64(old) / np.float64(new))
    kb, vb, ks, vs = (gpu.DeviceBuffer(n) for n in gpu.kv8_bytes(1, bt, 1, dim))
    cache = gpu.kv8_cache(kb, vb, ks, vs, 1, bt, 1, dim)
    table, zero = dev(gpu, i32([0])), dev(gpu, i32([0]))
    for rows_, at in ((first, 0), (last, held)):
        b = gpu.DeviceBuffer.from_numpy(rows_)
        gpu.kv8_append(cache, table, 1, b, b, dev(gpu, i32([0, len(rows_)])), dev(gpu, i32([at])), 1, len(rows_))
    assert ks.to_numpy(np.float32, (1,))[0] == new and vs.to_numpy(np.float32, (1,))[0] == new
    k = kb.to_numpy(np.int8, (bt, dim))[:held].reshape(held, 1, dim)
    v = vb.to_numpy(np.int8, (bt // 16, dim, 16)).transpose(0, 2, 1).reshape(bt, dim)[:held].reshape(held, 1, dim)
    assert np.array_equal(k, want) and np.array_equal(v, want)


@pytest.mark.parametrize("dtype,H,G,dim", [("f32", 4, 1, 64), ("bf16", 8, 1, 128), ("f16", 6, 2, 100), ("f32", 12, 12, 33)])
def test_chunks_joined_in_a_cluster(gpu, dtype, H, G, dim):
    """Up to eight chunks, of which a sequence needs none, one, some or all; the same bits each time, recorded too, for other
    lengths, and beside a length that is refused."""
    rng = np.random.default_rng(15)
    lengths, bt, top = [1500, 129, 0, 128, 700, 1], 16, 1700
    table, blocks = make_table([top] * len(lengths), bt, rng)
    c64 = Cache64(blocks, bt, G, dim, rng)
    for w in range(2):
        c64.s[w] *= (2.0 ** rng.integers(-4, 3, c64.s[w].shape)).astype(np.float32)
    dc = DeviceCache(gpu, c64)
    q = rows(rng, len(lengths), H, dim, dtype)
    scale = dim ** -0.5

    def right(got, lengths):
        ref = reference(c64, table, q, lengths, scale)
        assert bool(((got.double() - ref).abs() <= attention_tolerance(c64, table, lengths, q, scale, dtype, ref)).all())
    got = attention(gpu, dc, table, q, lengths, scale, dtype, max_len=top)
    right(got, lengths)
    out = torch.zeros_like(got)
    b = [dev(gpu, t) for t in (torch.from_numpy(table), q, out, i32(lengths))]
    with gpu.Recording() as rec:
        gpu.attn_kv8(dc.handle, b[0], table.shape[1], b[1], b[2], b[3], len(lengths), top, H, dtype=code(gpu, dtype))
    rec.replay(3)
    assert torch.equal(back(gpu, b[2], out), got)
    other = [0, 1700, 300, 1025, 256, 899]
    b[3].upload(np.array(other, np.int32))
    rec.replay(1)
    right(back(gpu, b[2], out), other)
    b[2].upload(torch.full_like(out, 3.0).view(torch.uint8).numpy())
    b[3].upload(np.array(other[:4] + [top + 1, 899], np.int32))
    rec.replay(1)
    last = back(gpu, b[2], out)
    with pytest.raises(gpu.SimpGpuError):
        gpu.check(gpu.lib().simp_gpu_check_device_status())
    assert bool((last[4] == 3.0).all())
    right(torch.where((torch.arange(6) == 4)[:, None, None], torch.zeros_like(last), last), other[:4] + [0, 899])
    rec.close()


def test_what_lies_behind_a_sequence_is_not_read(gpu):
    """Table entries behind the last block are garbage, scales of blocks in no sequence are NaN, max_len is larger than any
    length: no influence, nothing reported."""
    rng = np.random.default_rng(6)
    lengths, bt, dim = [40, 16, 1, 0], 16, 64
    table, blocks = make_table(lengths, bt, rng, extra=3, width=9, fill=12345678)
    c64 = Cache64(blocks, bt, 1, dim, rng)
    used = set(table[table < blocks].tolist())
    for b in range(blocks):
        if b not in used:
            c64.s[0][b] = c64.s[1][b] = np.nan
    dc = DeviceCache(gpu, c64)
    q = rows(rng, 4, 4, dim, "bf16")
    got = attention(gpu, dc, table, q, lengths, 0.125, "bf16", max_len=9 * bt)
    clean = Cache64(blocks, bt, 1, dim)
    clean.q, clean.s = c64.q, [np.nan_to_num(s) for s in c64.s]
    ref = reference(clean, table, q, lengths, 0.125)
    assert bool(((got.double() - ref).abs() <= attention_tolerance(clean, table, lengths, q, 0.125, "bf16", ref)).all())
    assert bool((got[3] == 0).all())


def test_query_that_is_not_finite(gpu):
    """Its head is NaN, the other heads and sequences are as without it."""
    rng = np.random.default_rng(7)
    lengths, bt, dim = [100, 300], 32, 64
    table, blocks = make_table(lengths, bt, rng)
    dc = DeviceCache(gpu, Cache64(blocks, bt, 2, dim, rng))
    for dtype in ("f32", "bf16"):
        q = rows(rng, 2, 8, dim, dtype)
        clean = attention(gpu, dc, table, q, lengths, 0.125, dtype)
        for bad in (math.nan, math.inf, -math.inf):
            q2 = q.clone()
            q2[1, 5, 7] = bad
            got = attention(gpu, dc, table, q2, lengths, 0.125, dtype)
            assert bool(torch.isnan(got[1, 5]).all())
            got[1, 5] = clean[1, 5]
            assert torch.equal(got, clean)


def test_strided_queries_and_outputs(gpu):
    rng = np.random.default_rng(8)
    lengths, bt, dim, H = [70, 33, 5], 16, 64, 4
    table, blocks = make_table(lengths, bt, rng)
    dc = DeviceCache(gpu, Cache64(blocks, bt, 2, dim, rng))
    q = rows(rng, 3, H, dim, "f16")
    want = attention(gpu, dc, table, q, lengths, 0.125, "f16")
    wide = torch.full((3, H * dim + 5), 3.0, dtype=torch.float16)
    wide[:, :H * dim] = q.reshape(3, -1)
    out = torch.full((3, H * dim + 9), 7.0, dtype=torch.float16)
    bo = dev(gpu, out)
    gpu.attn_kv8(dc.handle, dev(gpu, torch.from_numpy(table)), table.shape[1], dev(gpu, wide), bo, dev(gpu, i32(lengths)), 3, 70, H,
                 q_stride=H * dim + 5, out_stride=H * dim + 9, dtype=gpu.F16)
    got = back(gpu, bo, out)
    assert torch.equal(got[:, :H * dim].reshape(3, H, dim), want) and bool((got[:, H * dim:] == 7.0).all())
