"""GPU: penalties, biases, masks and the greedy choice.  The f32 arithmetic is a fixed sequence of single roundings, so results
are compared bit for bit with the same sequence in numpy (and to 64 bits in test_against_64_bits)."""
import numpy as np
import pytest
import torch

from serving_util import TYPES, back, code, dev, half_ulp, i32, offsets

pytestmark = pytest.mark.gpu


def make(seed, rows, vocab, dtype, history, biases, mask):
    rng = np.random.default_rng(seed)
    c = {"rows": rows, "vocab": vocab, "dtype": dtype}
    c["x"] = torch.from_numpy(rng.standard_normal((rows, vocab)) * 4).to(TYPES[dtype])
    c["lens"] = [int(rng.integers(0, history + 1)) for _ in range(rows)] if history is not None else None
    if history is not None:
        ids = (rng.random(sum(c["lens"])) ** 2 * vocab).astype(np.int32)
        ids[::11] = rng.choice([-1, vocab, 2 ** 31 - 1, -2 ** 31], ids[::11].shape)      # padding and the like: ignored
        c["ids"] = ids
        c["rep"], c["freq"], c["pres"] = (rng.uniform(a, b, rows).astype(np.float32) for a, b in ((0.8, 1.6), (-0.2, 0.7), (-0.3, 0.6)))
    c["nb"] = [int(rng.integers(0, biases + 1)) for _ in range(rows)] if biases is not None else None
    if biases is not None:
        c["bid"] = rng.integers(-2, vocab + 2, sum(c["nb"])).astype(np.int32)             # repeats among them: the last counts
        c["bval"] = (rng.standard_normal(sum(c["nb"])) * 3).astype(np.float32)
    words = (vocab + 31) // 32
    c["mask"] = rng.integers(0, 2 ** 32, (1 if mask == "one" else rows, words), dtype=np.uint64).astype(np.uint32) if mask else None
    return c


def expected(c, dt=np.float32):
    """The definition, operation by operation, in dt."""
    R, V = c["rows"], c["vocab"]
    x = c["x"].float().numpy().astype(dt)
    off = np.concatenate([[0], np.cumsum(c["lens"])]) if c["lens"] is not None else None
    boff = np.concatenate([[0], np.cumsum(c["nb"])]) if c["nb"] is not None else None
    for r in range(R):
        if off is not None:
            ids = c["ids"][off[r]:off[r + 1]]
            ids = ids[(ids >= 0) & (ids < V)]
            n = np.bincount(ids, minlength=V).astype(dt)
            hit = n > 0
            rep, f, p = dt(c["rep"][r]), dt(c["freq"][r]), dt(c["pres"][r])
            y = np.where(x[r] > 0, x[r] / rep, x[r] * rep)
            y = y - (f * n + p)
            x[r] = np.where(hit, y, x[r])
        if boff is not None:
            add = {int(t): v for t, v in zip(c["bid"][boff[r]:boff[r + 1]], c["bval"][boff[r]:boff[r + 1]]) if 0 <= t < V}
            for t, v in add.items():
                x[r, t] = x[r, t] + dt(v)
        if c["mask"] is not None:
            m = c["mask"][r if len(c["mask"]) > 1 else 0]
            bits = (m[:, None] >> np.arange(32, dtype=np.uint32)) & 1
            x[r, bits.reshape(-1)[:V] == 0] = -np.inf
    return x


def greedy(out):
    """Lowest index of the largest value; -1 where nothing is above -infinity; NaN passed over."""
    x = out.float().numpy()
    x = np.where(np.isnan(x), -np.inf, x)
    return np.where(x.max(1) == -np.inf, -1, x.argmax(1)).astype(np.int32)


def rules(gpu, c):
    keep, k = [], {}

    def put(name, arr):
        keep.append(gpu.DeviceBuffer.from_numpy(arr))
        k[name] = keep[-1]
    if c["lens"] is not None:
        put("tokens", c["ids"])
        put("token_offsets", offsets(c["lens"]).numpy())
        k["n_tokens"] = len(c["ids"])
        for n, m in (("repetition", "rep"), ("frequency", "freq"), ("presence", "pres")):
            put(n, c[m])
    if c["nb"] is not None:
        put("bias_tokens", c["bid"])
        put("bias_values", c["bval"])
        put("bias_offsets", offsets(c["nb"]).numpy())
        k["n_bias"] = len(c["bid"])
    if c["mask"] is not None:
        put("allowed", c["mask"])
        k["allowed_stride"] = c["mask"].shape[1] if len(c["mask"]) > 1 or c["rows"] == 1 else 0
    return gpu.logits_rules(**k), keep


def run(gpu, c, inplace=False, argmax=True):
    r, keep = rules(gpu, c)
    bx = dev(gpu, c["x"])
    bo = bx if inplace else dev(gpu, torch.full_like(c["x"], 7.0))
    best = gpu.DeviceBuffer.from_numpy(np.full(c["rows"], -7, np.int32))
    gpu.logits_process(bx, bo, c["rows"], c["vocab"], r, argmax=best if argmax else None, dtype=code(gpu, c["dtype"]))
    out = back(gpu, bo, c["x"])
    gpu.check(gpu.lib().simp_gpu_check_device_status())
    return out, best.to_numpy(np.int32, c["rows"])


def equal(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=1e30, posinf=2e30, neginf=-2e30), torch.nan_to_num(b.float(), nan=1e30, posinf=2e30, neginf=-2e30))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,history,biases,mask", [
    (1, 1, 3, 1, None), (1, 32000, 500, 20, "rows"), (3, 31, 40, 5, "rows"), (5, 33, 10, None, "one"), (2, 1023, None, 9, None), (4, 1025, 100, None, None),
    (7, 50001, 3000, 300, "rows"), (40, 4099, 50, 3, "one"), (130, 8191, 200, 10, "rows"), (2, 128256, 5000, 50, "rows"), (3, 100, None, None, "rows"), (6, 777, None, None, None),
    (2, 5, 0, 0, None)])
def test_bit_for_bit(gpu, dtype, rows, vocab, history, biases, mask):
    c = make(rows * 7 + vocab, rows, vocab, dtype, history, biases, mask)
    want = torch.from_numpy(expected(c)).to(TYPES[dtype])
    for inplace in (False, True):
        out, best = run(gpu, c, inplace)
        assert equal(out, want), f"{(out != want).sum()} logits differ"
        assert np.array_equal(best, greedy(want))
    out, best = run(gpu, c, argmax=False)
    assert equal(out, want) and bool((best == -7).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_against_64_bits(gpu, dtype):
    """Four f32 roundings, each relative to a value no larger than sum of magnitudes, and one to the type."""
    c = make(5, 6, 5000, dtype, 800, 40, "rows")
    ref = expected(c, np.float64)
    out, _ = run(gpu, c)
    fine = np.isfinite(ref)
    big = np.abs(c["x"].double().numpy()) * 1.6 + 0.7 * 800 + 0.6 + 12
    err = np.abs(out.double().numpy() - np.where(fine, ref, 0))
    assert np.array_equal(fine, np.isfinite(out.double().numpy()))
    assert np.all(err[fine] <= (4 * 2.0 ** -24 * big + half_ulp(TYPES[dtype]) * np.abs(np.where(fine, ref, 0)) * 1.001)[fine])


def test_not_finite_ties_and_nothing_allowed(gpu):
    x = torch.zeros(8, 3001)
    x[0, [5, 17, 2999]] = 4.0                      # a tie: the lowest
    x[1] = -np.inf
    x[1, 2000] = -1e38                             # the only one above -infinity
    x[2] = -np.inf                                 # nothing
    x[3] = np.nan                                  # nothing but NaN
    x[4, 7] = np.nan
    x[4, 9] = 1.0                                  # NaN is passed over
    x[5, 100] = np.inf
    x[6] = -0.0
    x[6, 50] = 0.0                                 # -0 and 0 are equal: the lowest
    x[7] = torch.linspace(-1, 1, 3001)             # its mask allows nothing
    c = {"rows": 8, "vocab": 3001, "dtype": "f32", "x": x, "lens": None, "nb": None}
    c["mask"] = np.full((8, 94), 0xffffffff, np.uint32)
    c["mask"][7] = 0
    out, best = run(gpu, c)
    want = x.clone()
    want[7] = -np.inf
    assert equal(out, want)
    assert best.tolist() == [5, 2000, -1, -1, 9, 100, 0, -1]
    out, again = run(gpu, c)                       # the scratch is as it was
    assert np.array_equal(best, again)


@pytest.mark.parametrize("dtype,first,pad,ofirst", [("f32", 1, 3, 0), ("f32", 2, 0, 2), ("bf16", 3, 5, 1), ("f16", 7, 8, 7)])
def test_rows_a_stride_apart_at_any_alignment(gpu, dtype, first, pad, ofirst):
    t, es, R, V = TYPES[dtype], TYPES[dtype].itemsize, 5, 4321
    c = make(9, R, V, dtype, 60, 8, "rows")
    stride = V + pad
    flat = torch.full((first + R * stride + 64,), 9.0, dtype=t)
    flat[first:first + R * stride].view(R, stride)[:, :V] = c["x"]
    oflat = torch.full((ofirst + R * stride + 64,), 7.0, dtype=t)
    r, keep = rules(gpu, c)
    bx, bo = dev(gpu, flat), dev(gpu, oflat)
    best = gpu.DeviceBuffer(4 * R)
    gpu.logits_process(bx.offset(first * es), bo.offset(ofirst * es), R, V, r, argmax=best, row_stride=stride, dtype=code(gpu, dtype))
    got = back(gpu, bo, oflat)
    want = torch.from_numpy(expected(c)).to(t)
    inside = got[ofirst:ofirst + R * stride].view(R, stride)
    assert equal(inside[:, :V], want) and bool((inside[:, V:] == 7.0).all())
    assert bool((got[:ofirst] == 7.0).all()) and bool((got[ofirst + R * stride:] == 7.0).all())
    assert np.array_equal(best.to_numpy(np.int32, R), greedy(want))


def test_bad_offsets_are_reported_and_that_list_skipped(gpu):
    c = make(3, 3, 500, "f32", 20, 4, None)
    for name, bad in (("lens", [0, 5, 3, 9]), ("lens", [0, 1, 2, 10 ** 6]), ("nb", [-1, 0, 1, 2])):
        r, keep = rules(gpu, c)
        b = gpu.DeviceBuffer.from_numpy(np.array(bad, np.int32))
        if name == "lens":
            r.token_offsets = b.ptr
        else:
            r.bias_offsets = b.ptr
        bx = dev(gpu, c["x"])
        gpu.logits_process(bx, bx, 3, 500, r)
        with pytest.raises(gpu.SimpGpuError, match="out of range"):
            gpu.check(gpu.lib().simp_gpu_check_device_status())
    gpu.check(gpu.lib().simp_gpu_check_device_status())


def test_recorded(gpu):
    c = make(4, 20, 32000, "f32", 300, 10, "rows")
    r, keep = rules(gpu, c)
    bx, bo, best = dev(gpu, c["x"]), dev(gpu, c["x"]), gpu.DeviceBuffer(80)
    call = lambda: gpu.logits_process(bx, bo, 20, 32000, r, argmax=best)
    call()
    with gpu.Recording() as rec:
        call()
    bo.zero()
    best.zero()
    rec.replay(3)
    want = torch.from_numpy(expected(c))
    assert equal(back(gpu, bo, c["x"]), want) and np.array_equal(best.to_numpy(np.int32, 20), greedy(want))
    rec.close()


@pytest.mark.parametrize("rows,vocab,biases", [(1, 9000, 20000), (40, 128256, 9000)])
def test_long_lists(gpu, rows, vocab, biases):
    """More biases than the usual path takes, many for the same token; histories longer than a thread keeps at hand."""
    c = make(11, rows, vocab, "f32", 6000, 10, "rows")
    rng = np.random.default_rng(12)
    c["nb"] = [biases - 7 * r for r in range(rows)]
    c["bid"] = rng.integers(0, vocab, sum(c["nb"])).astype(np.int32)
    c["bval"] = rng.standard_normal(sum(c["nb"])).astype(np.float32)
    want = torch.from_numpy(expected(c))
    out, best = run(gpu, c)
    assert equal(out, want) and np.array_equal(best, greedy(want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,history,biases", [(300, 8193, 4000, 40), (150, 16400, 300, 600), (2, 3000, 9000, 4)])
def test_rows_of_long_histories(gpu, dtype, rows, vocab, history, biases):
    """Histories with more different tokens in a block's slice than it lists, and rows with fewer, in long and short slices."""
    c = make(rows + vocab, rows, vocab, dtype, history, biases, "one")
    want = torch.from_numpy(expected(c)).to(TYPES[dtype])
    for inplace in (False, True):
        out, best = run(gpu, c, inplace)
        assert equal(out, want), f"{(out != want).sum()} logits differ"
        assert np.array_equal(best, greedy(want))
