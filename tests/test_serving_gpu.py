"""GPU: the serving ops used together, as a host would: prompts of a batch through attention into the 8-bit cache, a second
prompt that goes on behind the first (its cached rows read back), then single tokens over the cache and the rules on their
logits.  Every step is compared with 64-bit arithmetic on the same inputs."""
import math

import numpy as np
import pytest
import torch

from serving_util import TYPES, Cache64, DeviceCache, attend64, back, code, dev, half_ulp, i32, make_table, offsets, prompt_tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,H,G,D,bt", [("f32", 12, 12, 64, 32), ("bf16", 8, 2, 128, 64), ("f16", 8, 2, 64, 16), ("f32", 4, 4, 100, 16)])
def test_prompt_then_tokens(gpu, dtype, H, G, D, bt):
    t, rng, vocab = TYPES[dtype], np.random.default_rng(D), 4001
    first, second, steps = [70, 33, 128], [20, 0, 45], 5
    n, scale = len(first), D ** -0.5
    r = lambda rows, heads: torch.from_numpy(rng.standard_normal((rows, heads, D))).to(t)
    table, blocks = make_table([a + b + steps for a, b in zip(first, second)], bt, rng)
    c64 = Cache64(blocks, bt, G, D)
    dc = DeviceCache(gpu, c64)
    dt, width, ty = dev(gpu, torch.from_numpy(table)), table.shape[1], code(gpu, dtype)
    split = lambda x, lens: list(torch.split(x, lens))

    def prompt(q, k, v, nq, nk):
        out = torch.zeros_like(q)
        b = [dev(gpu, x) for x in (q, k, v, out, offsets(nq), offsets(nk))]
        gpu.attn_prompt(*b, n, q.shape[0], k.shape[0], H, G, D, dtype=ty)
        got = back(gpu, b[3], out)
        for s, (a, x, y, z) in enumerate(zip(split(got, nq), split(q, nq), split(k, nk), split(v, nk))):
            ref = attend64(x, y, z, scale)
            if len(x):
                assert bool(((a.double() - ref).abs() <= prompt_tolerance(x, y, z, scale, len(y), t, dtype != "f32") + half_ulp(t) * ref.abs()).all()), s

    def append(k, v, lens, starts):
        b = [dev(gpu, x) for x in (k, v, offsets(lens), i32(starts))]
        gpu.kv8_append(dc.handle, dt, width, *b, n, k.shape[0], dtype=ty)
        gpu.sync()
        c64.append(table, list(zip(split(k.double(), lens), split(v.double(), lens))), starts)
        q, s = dc.contents()
        assert all(np.array_equal(q[w], c64.q[w]) and np.array_equal(s[w], c64.s[w]) for w in range(2))

    k1, v1 = r(sum(first), G), r(sum(first), G)
    prompt(r(sum(first), H), k1, v1, first, first)
    append(k1, v1, first, [0] * n)
    # the second prompt: what the cache holds, then its own rows
    both = [a + b for a, b in zip(first, second)]
    k2, v2 = r(sum(second), G), r(sum(second), G)
    kall, vall = torch.zeros(sum(both), G, D, dtype=t), torch.zeros(sum(both), G, D, dtype=t)
    bk, bv = dev(gpu, torch.zeros(sum(first), G, D, dtype=t)), dev(gpu, torch.zeros(sum(first), G, D, dtype=t))
    gpu.kv8_read(dc.handle, dt, width, bk, bv, dev(gpu, offsets(first)), dev(gpu, i32([0] * n)), n, sum(first), dtype=ty)
    old_k, old_v = split(back(gpu, bk, torch.zeros(sum(first), G, D, dtype=t)), first), split(back(gpu, bv, torch.zeros(sum(first), G, D, dtype=t)), first)
    kall = torch.cat([x for pair in zip(old_k, split(k2, second)) for x in pair])
    vall = torch.cat([x for pair in zip(old_v, split(v2, second)) for x in pair])
    prompt(r(sum(second), H), kall, vall, second, both)
    append(k2, v2, second, first)
    # tokens
    texts = [list(rng.integers(0, vocab, 10)) for _ in range(n)]
    head = torch.from_numpy(rng.standard_normal((H * D, vocab)) * 0.05).float()
    for step in range(steps):
        lens = [b + step + 1 for b in both]
        k, v, q = r(n, G), r(n, G), r(n, H)
        append(k, v, [1] * n, [x - 1 for x in lens])
        out = torch.zeros_like(q)
        bo = dev(gpu, out)
        gpu.attn_kv8(dc.handle, dt, width, dev(gpu, q), bo, dev(gpu, i32(lens)), n, max(lens), H, dtype=ty)
        got = back(gpu, bo, out)
        ref = torch.cat([attend64(q[s:s + 1], torch.from_numpy(c64.values(table[s], lens[s], 0)), torch.from_numpy(c64.values(table[s], lens[s], 1)), scale) for s in range(n)])
        # largest |value| is below 6; the bound of the cache attention's own tests, rounded up
        assert float(((got.double() - ref).abs() - half_ulp(t) * ref.abs()).max()) <= (2e-5 if dtype == "f32" else 6e-3)
        logits = got.float().reshape(n, -1) @ head
        history = np.concatenate(texts).astype(np.int32)
        rules = gpu.logits_rules(tokens=(a := gpu.DeviceBuffer.from_numpy(history)), token_offsets=(b := gpu.DeviceBuffer.from_numpy(offsets([len(x) for x in texts]).numpy())),
                                 n_tokens=len(history), presence=(c := gpu.DeviceBuffer.from_numpy(np.full(n, 1e4, np.float32))))
        bl, best = dev(gpu, logits), gpu.DeviceBuffer(4 * n)
        gpu.logits_process(bl, bl, n, vocab, rules, argmax=best)
        tokens = best.to_numpy(np.int32, n)
        for s in range(n):      # with such a penalty no token comes twice
            free = logits[s].clone()
            free[torch.tensor(texts[s], dtype=torch.long)] = -math.inf
            assert int(tokens[s]) == int(free.argmax())
            texts[s].append(int(tokens[s]))
    gpu.check(gpu.lib().simp_gpu_check_device_status())


def test_calls_one_behind_the_other(gpu):
    """Steps enqueued without a wait between them (each launch may begin before the one before it has ended) give the bits of
    the same steps with a wait after each; recorded and replayed too."""
    rng, H, G, D, bt, n, steps, vocab = np.random.default_rng(3), 8, 2, 128, 32, 3, 12, 5000
    lens = [100, 7, 63]
    table, blocks = make_table([x + steps for x in lens], bt, rng)
    r = lambda *s: torch.from_numpy(rng.standard_normal(s)).to(torch.bfloat16)
    k, v, q = r(steps, n, G, D), r(steps, n, G, D), r(steps, n, H, D)
    dt, off = dev(gpu, torch.from_numpy(table)), dev(gpu, offsets([1] * n))
    bk, bv, bq = dev(gpu, k), dev(gpu, v), dev(gpu, q)
    starts = [dev(gpu, i32([x + s for x in lens])) for s in range(steps)]
    now = [dev(gpu, i32([x + s + 1 for x in lens])) for s in range(steps)]
    fill = Cache64(blocks, bt, G, D, rng)
    rules = gpu.logits_rules(tokens=(h := gpu.DeviceBuffer.from_numpy(np.arange(n * 9, dtype=np.int32))), token_offsets=(o := dev(gpu, offsets([9] * n))), n_tokens=9 * n,
                             presence=(p := gpu.DeviceBuffer.from_numpy(np.full(n, 0.5, np.float32))))

    def run(wait, record=False):
        dc = DeviceCache(gpu, fill)
        out, back_k, back_v = gpu.DeviceBuffer(steps * n * H * D * 2), gpu.DeviceBuffer(steps * n * G * D * 2), gpu.DeviceBuffer(steps * n * G * D * 2)
        best = gpu.DeviceBuffer(steps * n * 4)
        best.zero()

        def all_steps():
            for s in range(steps):
                gpu.kv8_append(dc.handle, dt, table.shape[1], bk.offset(s * n * G * D * 2), bv.offset(s * n * G * D * 2), off, starts[s], n, n, dtype=gpu.BF16)
                gpu.attn_kv8(dc.handle, dt, table.shape[1], bq.offset(s * n * H * D * 2), out.offset(s * n * H * D * 2), now[s], n, max(lens) + steps, H, dtype=gpu.BF16)
                gpu.kv8_read(dc.handle, dt, table.shape[1], back_k.offset(s * n * G * D * 2), back_v.offset(s * n * G * D * 2), off, starts[s], n, n, dtype=gpu.BF16)
                # the attention's output taken for logits: [n, H * D] bf16, in place
                gpu.logits_process(out.offset(s * n * H * D * 2), out.offset(s * n * H * D * 2), n, H * D, rules, argmax=best.offset(s * n * 4), dtype=gpu.BF16)
                if wait:
                    gpu.sync()
        if record:
            with gpu.Recording() as rec:
                all_steps()
            rec.replay(1)
            gpu.sync()
            rec.close()
        else:
            all_steps()
        return [b.to_numpy(np.uint8, b.nbytes).copy() for b in (out, back_k, back_v, best)] + [x.copy() for x in dc.contents()[0]]

    want = run(True)
    for _ in range(5):
        assert all(np.array_equal(a, b) for a, b in zip(run(False), want))
    assert all(np.array_equal(a, b) for a, b in zip(run(False, record=True), want))


def test_first_call_inside_a_recording():
    """In a new process: what needs scratch says so, prompt attention does without."""
    import subprocess
    import sys
    import os
    code_ = '''
import numpy as np, torch, sys
sys.path.insert(0, "tests")
import simplang_b200 as sg
from serving_util import attend64, back, dev, offsets, Cache64, DeviceCache, i32
sg.init(0)
g = torch.Generator().manual_seed(0)
q = torch.randn(50, 2, 64, generator=g)
out = torch.zeros_like(q)
b, bo, off = dev(sg, q), dev(sg, out), dev(sg, offsets([50]))
c = Cache64(8192 // 16, 16, 1, 64)
dc = DeviceCache(sg, c)
table = dev(sg, torch.arange(512, dtype=torch.int32))
ln, qq, oo = dev(sg, i32([4000])), dev(sg, q[:1, :1]), dev(sg, q[:1, :1])
lg, best = dev(sg, torch.zeros(1, 40000)), sg.DeviceBuffer(16)
codes = []
with sg.Recording() as rec:
    sg.attn_prompt(b, b, b, bo, off, None, 1, 50, 50, 2, 2, 64)
    for call in (lambda: sg.attn_kv8(dc.handle, table, 512, qq, oo, ln, 1, 8192, 1), lambda: sg.logits_process(lg, lg, 1, 40000, sg.logits_rules(), argmax=best)):
        try:
            call()
            codes.append(0)
        except sg.SimpGpuError as e:
            codes.append(e.code)
rec.replay(1)
got = back(sg, bo, out)
ref = attend64(q, q, q, 0.125)
assert codes == [-4, -4], codes
assert float((got.double() - ref).norm() / ref.norm()) < 1e-5
rec.close()
sg.check(sg.lib().simp_gpu_check_device_status())
print("fine")
'''
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code_], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


def test_places_beyond_32_bits(gpu):
    """Element offsets above 2^31: blocks at the far end of a large cache, rows at the far end of large tensors."""
    L = gpu.lib()
    rng = np.random.default_rng(5)
    # cache of 2.3 GB per side
    G, D, bt, blocks = 8, 128, 64, 35000
    kb, vb, sk, sv = gpu.kv8_bytes(blocks, bt, G, D)
    bufs = [gpu.DeviceBuffer(x) for x in (kb, vb, sk, sv)]
    handle = gpu.kv8_cache(*bufs, blocks, bt, G, D)
    table = np.array([[blocks - 1, 0, blocks - 2]], np.int32)
    k, v, q = (torch.from_numpy(rng.standard_normal((150, h, D))).float() for h in (G, G, G))
    t, off, st = dev(gpu, torch.from_numpy(table)), dev(gpu, offsets([150])), dev(gpu, i32([0]))
    gpu.kv8_append(handle, t, 3, dev(gpu, k), dev(gpu, v), off, st, 1, 150)
    c64 = Cache64(3, bt, G, D)
    local = np.array([[2, 0, 1]])
    c64.append(local, [(k.double(), v.double())], [0])
    ok_, ov_ = dev(gpu, torch.zeros_like(k)), dev(gpu, torch.zeros_like(v))
    gpu.kv8_read(handle, t, 3, ok_, ov_, off, st, 1, 150)
    for w, b in enumerate((ok_, ov_)):
        want = c64.values(local[0], 150, w)
        assert np.all(np.abs(back(gpu, b, k).double().numpy() - want) <= 2.0 ** -23 * np.abs(want))
    bo = dev(gpu, torch.zeros(1, G, D))
    gpu.attn_kv8(handle, t, 3, dev(gpu, q[:1]), bo, dev(gpu, i32([150])), 1, 192, G)
    ref = attend64(q[:1], torch.from_numpy(c64.values(local[0], 150, 0)), torch.from_numpy(c64.values(local[0], 150, 1)), D ** -0.5)
    assert float((back(gpu, bo, torch.zeros(1, G, D)).double() - ref).abs().max()) < 1e-5
    for b in bufs:
        b.free()
    # prompt attention: the last rows of q and out with more than 2^31 elements each
    H, D, rows, n = 32, 128, 530000, 100
    big_q, big_o = gpu.DeviceBuffer(rows * H * D * 2), gpu.DeviceBuffer(rows * H * D * 2)
    x, kv = torch.from_numpy(rng.standard_normal((n, H, D))).to(torch.bfloat16), torch.from_numpy(rng.standard_normal((2, n, 1, D))).to(torch.bfloat16)
    at = (rows - n) * H * D * 2
    raw = x.contiguous().view(torch.uint8).numpy().reshape(-1)
    gpu.check(L.simp_gpu_upload(big_q.offset(at), raw.ctypes.data, raw.nbytes))
    gpu.sync()
    gpu.attn_prompt(big_q, dev(gpu, kv[0]), dev(gpu, kv[1]), big_o, dev(gpu, i32([rows - n, rows])), dev(gpu, i32([0, n])), 1, rows, n, H, 1, D, dtype=gpu.BF16)
    got = np.empty(raw.nbytes, np.uint8)
    gpu.check(L.simp_gpu_download(got.ctypes.data, big_o.offset(at), raw.nbytes))
    got = torch.from_numpy(got).view(torch.bfloat16).reshape(n, H, D).double()
    ref = attend64(x, kv[0], kv[1], D ** -0.5)
    tol = prompt_tolerance(x, kv[0], kv[1], D ** -0.5, n, torch.bfloat16, True) + half_ulp(torch.bfloat16) * ref.abs()
    assert bool(((got - ref).abs() <= tol).all())
    big_q.free()
    big_o.free()
    # logits: 17000 rows of 128256 in place, a bias in the last one
    rows, vocab = 17000, 128256
    big = gpu.DeviceBuffer(rows * vocab * 4)
    big.zero()
    offs = np.zeros(rows + 1, np.int32)
    offs[-1] = 1
    rules = gpu.logits_rules(bias_tokens=(a := gpu.DeviceBuffer.from_numpy(np.array([vocab - 1], np.int32))), bias_values=(b := gpu.DeviceBuffer.from_numpy(np.array([2.5], np.float32))),
                             bias_offsets=(c := gpu.DeviceBuffer.from_numpy(offs)), n_bias=1)
    best = gpu.DeviceBuffer(rows * 4)
    gpu.logits_process(big, big, rows, vocab, rules, argmax=best)
    last = np.empty(vocab, np.float32)
    gpu.check(L.simp_gpu_download(last.ctypes.data, big.offset((rows - 1) * vocab * 4), vocab * 4))
    assert last[-1] == 2.5 and not last[:-1].any()
    tokens = best.to_numpy(np.int32, rows)
    assert tokens[-1] == vocab - 1 and not tokens[:-1].any()
    gpu.check(L.simp_gpu_check_device_status())
