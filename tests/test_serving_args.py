"""CPU: the batched serving ops refuse what they cannot serve before they touch a device (there is none here)."""
import ctypes as C

import pytest

P = 1 << 20    # a pointer that is never followed


@pytest.fixture()
def sg():
    import simplang_b200 as sg
    sg.lib()
    return sg


def refused(sg, code, text, fn, *args, **more):
    with pytest.raises(sg.SimpGpuError, match=text) as e:
        fn(*args, **more)
    assert e.value.code == code


ARG, SHAPE = -1, -2


def prompt(sg, q=P, k=P, v=P, out=P, qo=P, ko=None, n=2, tq=10, tk=10, H=4, G=2, D=64, **more):
    sg.attn_prompt(q, k, v, out, qo, ko, n, tq, tk, H, G, D, **more)


@pytest.mark.parametrize("code,text,more", [
    (ARG, "dtype", dict(dtype=3)), (ARG, "negative", dict(n=-1)), (ARG, "negative", dict(tq=-1)), (SHAPE, "head_dim", dict(D=0)), (SHAPE, "head_dim", dict(D=129)),
    (SHAPE, "heads", dict(G=3)), (SHAPE, "heads", dict(G=0)), (SHAPE, "heads", dict(H=0)), (SHAPE, "heads", dict(H=258, G=1)), (ARG, "null", dict(q=None)), (ARG, "null", dict(k=None)),
    (ARG, "null", dict(out=None)), (ARG, "null", dict(qo=None)), (SHAPE, "k_offsets", dict(tk=11)), (SHAPE, "stride", dict(q_stride=255)), (SHAPE, "stride", dict(kv_stride=1)),
    (SHAPE, "stride", dict(out_stride=-4)), (ARG, "misaligned", dict(q=P + 2)), (ARG, "misaligned", dict(out=P + 1, dtype=2)), (SHAPE, "too many", dict(tq=1 << 31, tk=1 << 31))])
def test_attn_prompt(sg, code, text, more):
    refused(sg, code, text, prompt, sg, **more)


def test_nothing_to_do_needs_no_device(sg):
    prompt(sg, q=None, k=None, v=None, out=None, qo=None, n=0, tq=0, tk=0)
    prompt(sg, n=3, tq=0, tk=0)
    c = cache(sg)
    sg.kv8_append(c, P, 4, None, None, None, None, 0, 0)
    sg.kv8_read(c, P, 4, None, None, None, None, 5, 0)
    sg.attn_kv8(c, P, 4, None, None, None, 0, 0, 4)
    sg.logits_process(None, None, 0, 100, sg.logits_rules())


def cache(sg, k=P, v=P, ks=P, vs=P, blocks=10, bt=16, G=2, D=64):
    return sg.kv8_cache(k, v, ks, vs, blocks, bt, G, D)


CACHES = [(SHAPE, "head_dim", dict(D=0)), (SHAPE, "head_dim", dict(D=200)), (SHAPE, "block_tokens", dict(bt=8)), (SHAPE, "block_tokens", dict(bt=48)), (SHAPE, "block_tokens", dict(bt=256)),
          (SHAPE, "blocks", dict(blocks=0)), (SHAPE, "blocks", dict(G=0)), (SHAPE, "blocks", dict(blocks=1 << 31)), (ARG, "null", dict(k=None)), (ARG, "null", dict(vs=None)), (ARG, "aligned", dict(k=P + 8)),
          (ARG, "aligned", dict(v=P + 1))]


@pytest.mark.parametrize("code,text,more", CACHES)
def test_caches(sg, code, text, more):
    c = cache(sg, **more)
    refused(sg, code, text, sg.kv8_append, c, P, 4, P, P, P, P, 1, 8)
    refused(sg, code, text, sg.kv8_read, c, P, 4, P, P, P, P, 1, 8)
    refused(sg, code, text, sg.attn_kv8, c, P, 4, P, P, P, 1, 8, 4)


def test_no_cache(sg):
    L = sg.lib()
    assert L.simp_gpu_kv8_append(None, P, 4, P, P, 0, P, P, 1, 8, 0) == ARG
    assert L.simp_gpu_kv8_read(None, P, 4, P, P, 0, P, P, 1, 8, 0) == ARG
    assert L.simp_gpu_attn_kv8(None, P, 4, P, P, 0, 0, P, 1, 8, 4, 1.0, 0) == ARG
    assert L.simp_gpu_logits_process(P, P, 1, 8, 0, None, None, 0) == ARG


@pytest.mark.parametrize("name", ["kv8_append", "kv8_read"])
def test_rows(sg, name):
    fn, c = getattr(sg, name), cache(sg)
    refused(sg, ARG, "dtype", fn, c, P, 4, P, P, P, P, 1, 8, dtype=-1)
    refused(sg, ARG, "negative", fn, c, P, 4, P, P, P, P, -1, 8)
    refused(sg, ARG, "negative", fn, c, P, 4, P, P, P, P, 1, -8)
    refused(sg, SHAPE, "table_stride", fn, c, P, 0, P, P, P, P, 1, 8)
    refused(sg, ARG, "null", fn, c, None, 4, P, P, P, P, 1, 8)
    refused(sg, SHAPE, "too many", fn, c, P, 4, P, P, P, P, 1, 1 << 31)
    for hole in range(4):
        a = [P] * 4
        a[hole] = None
        refused(sg, ARG, "null", fn, c, P, 4, *a, 1, 8)
    refused(sg, SHAPE, "kv_stride", fn, c, P, 4, P, P, P, P, 1, 8, kv_stride=127)
    refused(sg, ARG, "misaligned", fn, c, P, 4, P + 2, P, P, P, 1, 8)


def test_attn_kv8(sg):
    c, fn = cache(sg), sg.attn_kv8
    refused(sg, ARG, "dtype", fn, c, P, 4, P, P, P, 1, 8, 4, dtype=9)
    refused(sg, ARG, "negative", fn, c, P, 4, P, P, P, -1, 8, 4)
    refused(sg, ARG, "negative", fn, c, P, 4, P, P, P, 1, -8, 4)
    refused(sg, SHAPE, "heads", fn, c, P, 4, P, P, P, 1, 8, 3)
    refused(sg, SHAPE, "heads", fn, c, P, 4, P, P, P, 1, 8, 0)
    refused(sg, SHAPE, "max_len", fn, c, P, 4, P, P, P, 1, 65, 4)
    refused(sg, SHAPE, "2.30", fn, c, P, (1 << 27) - 1, P, P, P, 1, (1 << 30) + 1, 4)
    refused(sg, SHAPE, "65535", fn, c, P, 4, P, P, P, 70000, 8, 4)
    for hole in range(3):
        a = [P] * 3
        a[hole] = None
        refused(sg, ARG, "null", fn, c, P, 4, *a, 1, 8, 4)
    refused(sg, SHAPE, "stride", fn, c, P, 4, P, P, P, 1, 8, 4, q_stride=255)
    refused(sg, SHAPE, "stride", fn, c, P, 4, P, P, P, 1, 8, 4, out_stride=1)
    refused(sg, ARG, "misaligned", fn, c, P, 4, P + 1, P, P, 1, 8, 4)


def test_logits_process(sg):
    fn, r = sg.logits_process, sg.logits_rules
    refused(sg, ARG, "dtype", fn, P, P, 1, 8, r(), dtype=5)
    refused(sg, ARG, "negative", fn, P, P, -1, 8, r())
    refused(sg, SHAPE, "rows", fn, P, P, 1, 0, r())
    refused(sg, SHAPE, "rows", fn, P, P, 65536, 8, r())
    refused(sg, SHAPE, "rows", fn, P, P, 1, (1 << 30) + 1, r())
    refused(sg, ARG, "null", fn, None, P, 1, 8, r())
    refused(sg, ARG, "null", fn, P, None, 1, 8, r())
    refused(sg, SHAPE, "row_stride", fn, P, P, 1, 8, r(), row_stride=7)
    refused(sg, ARG, "misaligned", fn, P + 2, P, 1, 8, r())
    refused(sg, ARG, "go together", fn, P, P, 1, 8, r(tokens=P))
    refused(sg, ARG, "go together", fn, P, P, 1, 8, r(bias_tokens=P, bias_values=P))
    refused(sg, ARG, "need tokens", fn, P, P, 1, 8, r(repetition=P))
    refused(sg, ARG, "list", fn, P, P, 1, 8, r(tokens=P, token_offsets=P, n_tokens=-1))
    refused(sg, ARG, "list", fn, P, P, 1, 8, r(n_bias=1 << 31))
    refused(sg, SHAPE, "allowed_stride", fn, P, P, 1, 33, r(allowed=P, allowed_stride=1))


def test_lists_longer_than_the_kernel_counts(sg):
    fn, r, n = sg.logits_process, sg.logits_rules, (1 << 30) + 1
    refused(sg, ARG, "list", fn, P, P, 1, 8, r(tokens=P, token_offsets=P, n_tokens=n))
    refused(sg, ARG, "list", fn, P, P, 1, 8, r(bias_tokens=P, bias_values=P, bias_offsets=P, n_bias=n))


def test_sizes_of_a_cache(sg):
    assert sg.kv8_bytes(10, 16, 2, 100) == (10 * 16 * 2 * 128, 10 * 16 * 2 * 128, 80, 80)
    assert C.sizeof(sg.Kv8Cache) == 64 and C.sizeof(sg.LogitsRules) == 96
