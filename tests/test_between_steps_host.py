"""What the operators between two steps refuse, without a GPU: arguments the Python layer turns down, and those the C entries turn down before any CUDA call."""
import ctypes as C

import pytest
import torch

from blazr_b200 import seqops

f32, i32 = torch.float32, torch.int32


@pytest.fixture(scope="module")
def L():
    return seqops.lib()


def verify_args(**kw):
    d = dict(logits=torch.zeros(3, 10), start=torch.tensor([0, 2, 3], dtype=i32), drafts=torch.zeros(3, dtype=i32), accept_u=torch.zeros(3), sample_u=torch.zeros(2), temperature=torch.ones(2))
    d.update(kw)
    return d


@pytest.mark.parametrize("kw", [
    dict(logits=torch.zeros(3, 10, dtype=torch.bfloat16)), dict(logits=torch.zeros(30)), dict(logits=torch.zeros(10, 3).t()), dict(logits=torch.zeros(3, 0)), dict(start=torch.zeros(2, dtype=i32)),
    dict(start=torch.zeros(3, dtype=torch.int64)), dict(drafts=torch.zeros(4, dtype=i32)), dict(accept_u=torch.zeros(3, dtype=torch.float64)), dict(sample_u=torch.zeros(3)),
    dict(temperature=torch.ones(2, dtype=torch.float64)), dict(top_k=torch.zeros(2)), dict(top_p=torch.zeros(3)), dict(draft_probs=torch.zeros(2, 10)), dict(draft_probs=torch.zeros(10, 3).t()),
    dict(accepted=torch.zeros(3, dtype=i32)), dict(tokens=torch.zeros(2, dtype=i32)), dict(sample_u=torch.zeros(4)[::2]), {}], ids=lambda k: " ".join(k) or "no GPU")
def test_verify_drafts_refuses(L, kw):
    with pytest.raises(ValueError):
        seqops.verify_drafts(**verify_args(**kw))


def test_verify_drafts_c_refuses(L):
    p = C.c_void_p(16)
    call = lambda ld=10, R=3, V=10, start=p, B=2, scratch=p, n=1 << 20, q=None, ldq=10, logits=p: L.b200seq_verify_drafts(logits, ld, R, V, start, B, p, p, p, p, None, None, q, ldq, p, p,
                                                                                                                          scratch, n, None)
    for kw in (dict(R=-1), dict(V=0), dict(B=-1), dict(start=None), dict(logits=None), dict(ld=9), dict(q=p, ldq=9), dict(scratch=None), dict(n=8), dict(scratch=C.c_void_p(24)), dict(R=70000),
               dict(V=1 << 30, ld=1 << 30)):
        assert call(**kw) < 0, kw
        assert b"verify_drafts" in L.b200seq_last_error()
    assert call(B=0) == 0
    assert L.b200seq_verify_scratch_bytes(0, 10, 0) == 0 and L.b200seq_verify_scratch_bytes(3, 10, 1) > L.b200seq_verify_scratch_bytes(3, 10, 0) > 0


def step(T=2, B=2, mb=4, bs=16):
    return seqops.StepDesc(16, 16, 16, 16, 16, 16, T, B, mb, bs)


def layer(**kw):
    return seqops.attn_desc(4, 2, 64, 64, 0.125, gated=False, kv_shared=True, **kw)


@pytest.mark.parametrize("kw", [
    dict(proj=torch.zeros(2, 256, dtype=torch.bfloat16)), dict(proj=torch.zeros(1, 256)), dict(proj=torch.zeros(2, 255)), dict(proj=torch.zeros(256, 2).t()), dict(kpool=torch.zeros(5, 8, 2, 64)),
    dict(kpool=torch.zeros(5, 16, 4, 64)), dict(kpool=torch.zeros(5, 16, 2, 64, dtype=torch.float16)), dict(kpool=torch.zeros(5, 2, 600, dtype=torch.uint8)), dict(acc=torch.zeros(3, 4, 64)),
    dict(acc=torch.zeros(3, 2, 64, dtype=torch.float64)), dict(acc=torch.zeros(3, 2, 128)[:, :, ::2]), dict(acc=torch.zeros(0, 2, 64)), dict(last=-1), dict(max_keys=-1), {}],
    ids=lambda k: " ".join(k) or "no GPU")
def test_key_weights_refuses(L, kw):
    d = dict(proj=torch.zeros(2, 256), step=step(), d=layer(), kpool=torch.zeros(5, 16, 2, 64), acc=torch.zeros(3, 2, 64))
    d.update(kw)
    with pytest.raises(ValueError):
        seqops.key_weights(**d)


def test_key_weights_c_refuses(L):
    p = C.c_void_p(16)

    def call(d=None, st=None, ld=256, kpool=p, bits=32, acc=p, slots=3, room=64, last=0, max_keys=0, scratch=p, n=1 << 22):
        return L.b200seq_key_weights(p, ld, C.byref(st or step()), C.byref(d or layer()), kpool, bits, acc, slots, room, last, max_keys, scratch, n, None)
    for kw in (dict(kpool=None), dict(acc=None), dict(bits=8), dict(slots=0), dict(room=0), dict(last=-1), dict(max_keys=-1), dict(scratch=None), dict(n=3), dict(ld=255), dict(scratch=C.c_void_p(20)),
               dict(st=step(T=-1)), dict(st=step(mb=0)), dict(st=step(bs=0)), dict(bits=4, kpool=C.c_void_p(20)), dict(st=step(T=70000, B=70000), n=1 << 40)):
        assert call(**kw) < 0, kw
        assert b"key_weights" in L.b200seq_last_error(), kw
    pooled = layer(window=32, pool=4)
    pooled.kv_shared = 0
    assert call(d=pooled) == -2                                        # pooled blocks beside the keys
    wide = seqops.attn_desc(2, 2, 160, 160, 0.1, gated=False, kv_shared=True)
    assert call(d=wide, ld=320, bits=4) == -2
    latent = seqops.latent_attn_desc(4, 64, 16, 0.1, gated=False)
    assert call(d=latent, ld=4096) == -2
    assert call(st=step(T=0)) == 0 and call(st=step(B=0)) == 0


def evict_args(**kw):
    d = dict(kpools=[torch.zeros(6, 16, 2, 64)], vpools=[torch.zeros(6, 16, 2, 64)], accs=[torch.zeros(3, 2, 64)], slots=torch.zeros(1, dtype=i32), rows=torch.tensor([40], dtype=i32),
             table=torch.zeros(1, 3, dtype=i32), keep=20, first=2, recent=4)
    d.update(kw)
    return d


@pytest.mark.parametrize("kw", [
    dict(kpools=[], vpools=[], accs=[]), dict(vpools=[]), dict(accs=[]), dict(kpools=[torch.zeros(6, 16, 2, 64).half()]), dict(kpools=[torch.zeros(6, 2, 1280, dtype=torch.uint8)]),
    dict(kpools=[torch.zeros(6, 2, 999, dtype=torch.uint8)], vpools=[torch.zeros(6, 2, 640, dtype=torch.uint8)], block_size=16), dict(vpools=[torch.zeros(6, 8, 2, 64)]),
    dict(vpools=[torch.zeros(5, 16, 2, 64)]), dict(block_size=8), dict(accs=[torch.zeros(3, 4, 64)]), dict(accs=[torch.zeros(3, 2, 64).double()]), dict(keep=0), dict(first=-1), dict(recent=-1), dict(first=17),
    dict(slots=torch.zeros(2, dtype=i32)), dict(slots=torch.zeros(1)), dict(table=torch.zeros(3, dtype=i32)), dict(table=torch.zeros(2, 3, dtype=i32)), dict(table=torch.zeros(1, 3)),
    dict(to_table=torch.zeros(1, 0, dtype=i32)), dict(to_slots=torch.zeros(1)), dict(kept=torch.zeros(19, dtype=i32)), dict(kpools=[torch.zeros(6, 16, 2, 128)[..., ::2]]), {}],
    ids=lambda k: " ".join(k) or "no GPU")
def test_evict_keys_refuses(L, kw):
    with pytest.raises(ValueError):
        seqops.evict_keys(**evict_args(**kw))


def test_evict_keys_c_refuses(L):
    p = C.c_void_p(16)
    arr = (C.c_void_p * 1)(16)
    odd = (C.c_void_p * 1)(20)

    def call(pools=arr, layers=1, bits=32, bs=16, G=2, D=64, Gv=2, V=64, slots=3, room=64, slot=p, mb=3, to_mb=3, B=1, keep=20, first=2, recent=4, kept=p):
        return L.b200seq_evict_keys(pools, arr, arr, layers, bits, bs, G, D, Gv, V, slots, room, slot, p, p, mb, p, p, to_mb, B, keep, first, recent, kept, None)
    for kw in (dict(pools=None), dict(layers=-1), dict(bits=16), dict(bs=0), dict(G=0), dict(D=0), dict(V=0), dict(Gv=4), dict(slots=0), dict(room=0), dict(slot=None), dict(mb=0), dict(to_mb=0), dict(B=-1),
               dict(keep=0), dict(first=-1), dict(recent=-1), dict(first=10, recent=11), dict(first=2 ** 31 - 1, recent=2 ** 31 - 1), dict(kept=None), dict(bits=4, D=129), dict(bits=4, pools=odd), dict(B=65536),
               dict(G=256, Gv=256, B=256), dict(pools=(C.c_void_p * 1)(None))):
        assert call(**kw) < 0, kw
        assert b"evict_keys" in L.b200seq_last_error()
    assert call(layers=0) == 0 and call(B=0) == 0


def test_verify_drafts_refuses_tokens_over_drafts(L):
    p = C.c_void_p(16)
    for d, t in ((64, 64), (64, 72), (72, 64)):
        assert L.b200seq_verify_drafts(p, 10, 3, 10, p, 2, C.c_void_p(d), p, p, p, None, None, None, 10, p, C.c_void_p(t), p, 1 << 20, None) == -1
        assert b"share memory" in L.b200seq_last_error()


@pytest.mark.parametrize("k,v,a", [((64, 64), (128, 192), (256, 512)), ((64, 320), (128, 128), (256, 512)), ((64, 320), (64, 192), (256, 512)), ((64, 320), (128, 64), (256, 512)),
                                   ((64, 320), (128, 192), (256, 256))])
def test_evict_keys_refuses_what_is_given_twice(L, k, v, a):
    p, arr = C.c_void_p(16), lambda x: (C.c_void_p * 2)(*x)
    assert L.b200seq_evict_keys(arr(k), arr(v), arr(a), 2, 32, 16, 2, 64, 2, 64, 3, 64, p, p, p, 3, p, p, 3, 1, 20, 2, 4, p, None) == -1
    assert b"given twice" in L.b200seq_last_error()
