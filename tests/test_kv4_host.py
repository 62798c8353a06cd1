"""What the 4-bit cache, page copies and sampling rules refuse, and the page sizes, without a GPU: every refusal comes before anything is launched."""
import ctypes as C

import numpy as np
import pytest
import torch

import kv4_oracle as ref
from blazr_b200 import seqops as ops


def step(T=2, B=1, bs=16, blocks=4):
    p = 0x1000
    return ops.StepDesc(p, p, p, p, p, p, T, B, blocks, bs)


@pytest.mark.parametrize("D", [1, 32, 33, 64, 65, 80, 128])
def test_page_bytes(D):
    assert ops.kv4_page_bytes(16, 3, D) == 16 * 3 * ref.groups(D) * 20
    assert ops.kv4_page_bytes(5, 1, D) == 100 * ref.groups(D)


@pytest.mark.parametrize("args", [(0, 1, 64), (16, 0, 64), (16, 1, 0), (16, 1, 129), (-3, 1, 64)])
def test_no_such_pages(args):
    with pytest.raises(ValueError):
        ops.kv4_page_bytes(*args)


def test_the_restatement_round_trips():
    """layout of the oracle itself: what is put is what is got, places behind D stay empty"""
    rng = np.random.default_rng(0)
    for D, bs in ((128, 16), (80, 32), (33, 5), (3, 1)):
        for key in (True, False):
            x = rng.standard_normal((2 * bs, 2, D)).astype(np.float32)
            pool = np.zeros((3, 2, bs * ref.groups(D) * 20), np.uint8)
            slots = [(p, o) for p in (2, 0) for o in range(bs)]
            ref.put_rows(pool, bs, slots, x, key)
            np.testing.assert_allclose(ref.get_rows(pool, bs, slots, D, key), ref.held(x), rtol=1e-7, atol=1e-7)
            assert not pool[1].any()


def entry(name):
    return getattr(ops.lib(), "b200seq_" + name)


P = 0x1000   # an address that is never followed


def layer(**o):
    kw = dict(H=8, G=2, D=64, V=64)
    kw.update({k: o.pop(k) for k in list(o) if k in kw})
    d = ops.attn_desc(kw["H"], kw["G"], kw["D"], kw["V"], 1.0, gated=False, **{k: o.pop(k) for k in list(o) if k in ("chunk", "window", "pool", "keep_first")})
    for k, v in o.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("d,code", [(layer(D=129), -2), (layer(V=160), -2), (layer(window=32, pool=8), -2), (layer(G=1, latent_v=1), -2), (layer(ctx_rows=1), -2), (layer(kv_ld=640), -2),
                                    (layer(H=7), -1), (layer(D=0), -1), (layer(keep_first=2), -1), (layer(vg=3), -1)])
def test_layers_that_are_refused(d, code):
    st = step()
    assert entry("attn_kv4")(P, 1024, C.byref(st), C.byref(d), P, P, P, 0, None, 0, 0, None) == code
    if not d.kv_ld:
        assert entry("attn_prep_kv4")(P, 1024, C.byref(st), C.byref(d), P, P, None) == code


@pytest.mark.parametrize("st", [step(T=-1), step(B=-1), step(bs=0), step(blocks=-1), step(B=0), step(bs=1 << 17), ops.StepDesc(P, 0, P, P, P, P, 2, 1, 4, 16),
                                ops.StepDesc(P, P, P, P, P, 0, 2, 1, 4, 16)], ids=range(8))
def test_steps_that_are_refused(st):
    d = layer()
    assert entry("attn_kv4")(P, 1024, C.byref(st), C.byref(d), P, P, P, 0, None, 0, 0, None) < 0
    if st.B:
        assert entry("kv4_store")(P, 128, P, 128, 0, C.byref(st), 2, 64, 2, 64, P, P, None) < 0
        assert entry("kv4_load")(P, P, C.byref(st), 2, 64, 2, 64, P, 128, P, 128, None) < 0
        assert entry("attn_prep_kv4")(P, 1024, C.byref(st), C.byref(d), P, P, None) < 0


def test_arguments_that_are_refused():
    st, d = step(), layer()
    for bad in ((None, 1024, C.byref(st), C.byref(d), P, P, P, 0, None), (P, 1024, C.byref(st), C.byref(d), None, P, P, 0, None), (P, 1024, C.byref(st), C.byref(d), P, None, P, 0, None),
                (P, 1024, C.byref(st), C.byref(d), P, P, None, 0, None), (P, 1024, C.byref(st), C.byref(d), P, P, P, 1, None), (P, 1024, C.byref(st), C.byref(d), P + 8, P, P, 0, None),
                (P, 1024, None, C.byref(d), P, P, P, 0, None), (P, 1024, C.byref(st), None, P, P, P, 0, None)):
        assert entry("attn_kv4")(*bad[:-1], None, 0, 0, None) == -1
    for bad in ((P, 100, P, 128, 0, C.byref(st), 2, 64, 2, 64, P, P, None), (P, 128, P, 128, 7, C.byref(st), 2, 64, 2, 64, P, P, None), (P, 128, P, 128, 0, C.byref(st), 0, 64, 2, 64, P, P, None),
                (None, 128, P, 128, 0, C.byref(st), 2, 64, 2, 64, P, P, None), (P, 128, P, 128, 0, C.byref(st), 2, 64, 2, 64, P + 4, P, None)):
        assert entry("kv4_store")(*bad) == -1
    assert entry("kv4_store")(P, 1024, P, 128, 0, C.byref(st), 2, 129, 2, 64, P, P, None) == -2
    none = step(T=0)
    assert entry("attn_kv4")(P, 1024, C.byref(none), C.byref(d), P, P, P, 0, None, 0, 0, None) == 0
    assert entry("kv4_store")(None, 128, None, 128, 0, C.byref(none), 2, 64, 2, 64, P, P, None) == 0


def test_tensors_that_are_refused():
    st, d = step(), layer()
    kp = torch.zeros((4, 2, 640), dtype=torch.uint8)
    rows, out = torch.zeros(2, 1024), torch.zeros(2, 512)
    x = torch.zeros(2, 128)
    for call in (lambda: ops.attn_kv4(rows, st, d, kp.float(), kp, out), lambda: ops.attn_kv4(rows, st, d, kp[:, :1], kp, out), lambda: ops.attn_kv4(rows, st, d, kp[:, :, :320], kp, out),
                 lambda: ops.attn_kv4(rows.half(), st, d, kp, kp, out), lambda: ops.attn_kv4(rows[:1], st, d, kp, kp, out), lambda: ops.attn_kv4(rows[:, :500], st, d, kp, kp, out),
                 lambda: ops.attn_kv4(rows, st, d, kp, kp, out.half()), lambda: ops.attn_kv4(rows, st, d, kp, kp, out[:, :100]), lambda: ops.attn_kv4(rows, st, d, kp, kp, out[:1]),
                 lambda: ops.attn_kv4(rows, st, d, kp, kp, out, gate=rows[:, :4]), lambda: ops.attn_prep_kv4(rows[:, :600], st, d, kp, kp), lambda: ops.attn_kv4(rows, st, d, kp, kp, out),
                 lambda: ops.kv4_store(x, x.bfloat16(), st, kp, kp), lambda: ops.kv4_store(x.half(), x.half(), st, kp, kp), lambda: ops.kv4_store(x[:, :127], x, st, kp, kp),
                 lambda: ops.kv4_store(x[:1], x, st, kp, kp), lambda: ops.kv4_store(x.t(), x, st, kp, kp), lambda: ops.kv4_load(kp, kp, st, x.bfloat16(), x.bfloat16()),
                 lambda: ops.kv4_store(x, x, st, kp, kp)):
        with pytest.raises(ValueError):
            call()


def test_copies_that_are_refused():
    ptrs, size = (C.c_void_p * 1)(P), (C.c_int64 * 1)(64)
    call = lambda pairs, pages=6: entry("copy_pages")(ptrs, size, 1, pages, (C.c_int32 * (2 * len(pairs)))(*[x for p in pairs for x in p]), len(pairs), None)
    for pairs in ([(0, 1), (2, 1)], [(0, 1), (1, 2)], [(1, 2), (0, 1)], [(3, 3)], [(0, 6)], [(6, 0)], [(-1, 2)], [(2, -1)]):
        assert call(pairs) == -1, pairs
    assert call([(0, 0)], 0) == -1
    assert entry("copy_pages")(ptrs, size, 1, 6, None, 0, None) == 0
    assert entry("copy_pages")(None, None, 0, 6, None, 0, None) == 0
    assert entry("copy_pages")((C.c_void_p * 1)(None), size, 1, 6, None, 0, None) == -1
    with pytest.raises(ValueError):
        ops.copy_pages([torch.zeros(6, 4)], [(0, 1)])
    with pytest.raises(ValueError):
        ops.copy_pages([torch.zeros(6, 4), torch.zeros(5, 4)], [(0, 1)])


def test_logit_rules_that_are_refused():
    f = entry("process_logits")
    ok = [P, 100, 2, 100, P, P, 8, P, P, P, P, P, 8, P, 4, P, 100, None]
    for i, v in ((0, None), (1, 99), (2, -1), (3, 0), (4, None), (4, P + 4), (5, None), (6, -1), (7, None), (8, None), (9, None), (10, None), (11, None), (12, -1), (14, 3), (15, None), (16, 50)):
        a = list(ok)
        a[i] = v
        assert f(*a) == -1, (i, v)
    assert f(*(ok[:2] + [70000] + ok[3:])) == -2
    assert f(*(ok[:2] + [0] + ok[3:])) == 0
    x, r = torch.zeros(2, 100), torch.ones(2, 4)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    for call in (lambda: ops.process_logits(x.half(), r), lambda: ops.process_logits(x, r[:1]), lambda: ops.process_logits(x, r, x[:, :50]), lambda: ops.process_logits(x.t(), r),
                 lambda: ops.process_logits(x, r, mask=torch.zeros(2, 3, dtype=torch.int32)), lambda: ops.process_logits(x, r, mask=torch.zeros(2, 4)),
                 lambda: ops.process_logits(x, r, hist=i32(5).long(), hist_start=i32(3), hist_prompt=i32(2)), lambda: ops.process_logits(x, r, hist=i32(5), hist_start=i32(2), hist_prompt=i32(2)),
                 lambda: ops.process_logits(x, r, bias_ids=i32(5), bias_vals=torch.zeros(4), bias_start=i32(3)), lambda: ops.process_logits(x, r)):
        with pytest.raises(ValueError):
            call()
