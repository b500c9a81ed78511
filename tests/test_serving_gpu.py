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
