"""Operators of the serving path around a cache held in 4 bits, as cases that can be timed and checked one by one.

  store     keys and values of a step's tokens are quantised into the pages of their sequences, and read back as the values they stand for
  attend    attention of a step (single tokens, drafts to verify, prompt portions) over such pages
  copy      pages are copied inside every pool of a model (a forked request's last page, a compaction of the whole cache)
  logits    penalties for repeated tokens, biases, temperature and a grammar mask on rows of logits

A page holds for every head `block_size` rows; 32 neighbouring values of a row share a step s and a minimum m (both f16) and have a code of 4 bits each: a
value is m + s * code.  A row of D values is padded to P = 32, 64 or 128, NG = P / 32 groups.  Bytes of one head of a page: units of 16 rows, in each
first the rows' codes (P / 2 bytes a row), then the rows' (s, m) pairs (4 NG bytes a row).  Codes of a key row: 32-bit words [part c < 4][group g < NG],
eight values 32 g + 8 c + i in 4-bit fields from the lowest; of a value row: 16-bit words [part r < 8][group g < NG], four values 32 g + 4 r + i.

`own` chooses between the plain forms below (elementary torch operations in 32 bits) and the framework's calls.
"""
import math

import torch

DEV = "cuda:0"
own = False
BS = 16                     # tokens of a page: the engine's default
FIFTEENTH = float.fromhex("0x1.11111p-4")   # the 32-bit number below 1 / 15: a range of fifteen whole steps keeps its step


def listed():
    return [
        # one decoded token's keys and values enter the cache: the smallest call
        dict(name="store_1_token", kind="store", B=1, n=1, past=900, G=8, D=128, type="f32"),
        # two prompts of odd length enter the cache from 16-bit rows
        dict(name="store_2x2047_bf16", kind="store", B=2, n=2047, past=37, G=8, D=128, type="bf16"),
        # one sequence decodes behind a short context
        dict(name="attend_1_token", kind="attend", B=1, n=1, past=500, ragged=False, H=32, G=8, D=64, window=0, type="f32"),
        # 32 sequences decode behind contexts of 2000 to 4000 tokens
        dict(name="attend_32_sequences", kind="attend", B=32, n=1, past=4000, ragged=True, H=32, G=8, D=128, window=0, type="bf16"),
        # one sequence decodes behind a context of 128 k tokens
        dict(name="attend_131072_keys", kind="attend", B=1, n=1, past=131071, ragged=False, H=32, G=8, D=128, window=0, type="bf16"),
        # 16 sequences with five draft tokens each to verify
        dict(name="attend_16x5_drafts", kind="attend", B=16, n=5, past=1500, ragged=True, H=32, G=8, D=64, window=0, type="f32"),
        # a prompt of 2048 tokens
        dict(name="attend_2048_tokens", kind="attend", B=1, n=2048, past=0, ragged=False, H=32, G=8, D=128, window=0, type="bf16"),
        # a portion of odd length of a long prompt, windowed layer, 32-bit activations
        dict(name="attend_531_behind_5000", kind="attend", B=1, n=531, past=5000, ragged=False, H=32, G=8, D=64, window=2048, type="f32"),
        # four requests are forked: their partly filled last pages are copied in all pools of an eight-layer model
        dict(name="copy_4_pages", kind="copy", pools=16, pages=300, copied=4, G=8, D=128, bits=4),
        # a cache of 32-bit pages is compacted
        dict(name="copy_700_pages", kind="copy", pools=8, pages=1500, copied=700, G=8, D=64, bits=32),
        # 64 sampled sequences of a 128 k vocabulary, with long histories, biases and a grammar
        dict(name="logits_64_rows", kind="logits", R=64, V=128256, hist=4000, bias=300, mask=True),
        # one sequence of a 32 k vocabulary
        dict(name="logits_1_row", kind="logits", R=1, V=32000, hist=500, bias=0, mask=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "attend", "copy", "logits"])
    if kind == "store":
        B, D = rng.choice([1, 1, 2, 5]), rng.choice([64, 80, 128, 128])
        return dict(kind=kind, B=B, n=_log(rng, 1, 4096 // B), past=rng.randint(0, 2000), G=rng.choice([1, 2, 4, 8]), D=D, type=rng.choice(["f32", "bf16"]))
    if kind == "copy":
        bits = rng.choice([4, 32])
        pages = _log(rng, 30, 1500)
        return dict(kind=kind, pools=rng.randint(1, 16 if bits == 4 else 8), pages=pages, copied=_log(rng, 1, min(690, pages // 2 - 5)), G=rng.choice([2, 4, 8]), D=rng.choice([32, 64]), bits=bits)
    if kind == "logits":
        return dict(kind=kind, R=_log(rng, 1, 64), V=rng.choice([16384, 32000, 50257, 128256]), hist=_log(rng, 1, 4000), bias=rng.choice([0, 1, 50, 300]), mask=rng.random() < 0.5)
    H, G, D = rng.choice([(32, 8, 64), (32, 8, 128), (32, 4, 128), (16, 4, 64), (64, 8, 128), (16, 16, 80), (8, 1, 64)])
    form, kind = rng.choice(["decode", "decode", "drafts", "prompt", "prompt"]), "attend"
    window = rng.choice([0, 0, 0, 1024, 300])
    if form == "decode":
        B = _log(rng, 1, 64)
        return dict(kind=kind, B=B, n=1, past=_log(rng, 1, min(131071, 131072 // B)), ragged=True, H=H, G=G, D=D, window=window, type=rng.choice(["f32", "bf16"]))
    if form == "drafts":
        B = _log(rng, 1, 32)
        return dict(kind=kind, B=B, n=rng.randint(2, 9), past=_log(rng, 1, 65536 // B), ragged=True, H=H, G=G, D=D, window=window, type=rng.choice(["f32", "bf16"]))
    n = _log(rng, 17, 2048 if H < 64 else 1024)
    return dict(kind=kind, B=1, n=n, past=rng.choice([0, 0, _log(rng, 16, 400 if H == 64 else 1024)]) if n < 1024 else 0, ragged=False, H=H, G=G, D=D, window=window, type=rng.choice(["f32", "bf16"]))


# ---- inputs -----------------------------------------------------------------------------------------------------------------------
def _groups(D):
    return 1 if D <= 32 else 2 if D <= 64 else 4


def _pasts(c):
    """tokens that every sequence has in the cache: all the same, or spread evenly from half of it on"""
    B, past = c["B"], c["past"]
    return [past - ((i * 7919) % B * (past // 2)) // B if c.get("ragged") else past for i in range(B)]


def _pages(c):
    return [-(-(p + c["n"]) // BS) for p in _pasts(c)]


def _rand_pool(pages, G, NG, mean, g):
    """pages of random codes; steps and minima as values of unit spread (around a mean that differs from group to group, as keys have it) give them"""
    rows = pages * G * BS
    codes = torch.randint(0, 256, (rows, NG * 16), dtype=torch.uint8, device=DEV, generator=g)
    bits = torch.randint(70, 128, (rows, NG), device=DEV, generator=g).float()                 # seven significant bits: 64 .. 127
    step = (bits / 512).half()
    low = (mean * torch.randn(NG, device=DEV, generator=g) - 7.5 * step.float() + 0.1 * torch.randn((rows, NG), device=DEV, generator=g)).half()
    par = torch.stack([step, low], -1).contiguous().view(torch.uint8).reshape(rows, NG * 4)
    unit = torch.cat([codes.reshape(-1, BS * NG * 16), par.reshape(-1, BS * NG * 4)], 1)
    return unit.reshape(pages, G, BS * NG * 20).contiguous()


def _step(c, g):
    """int32 arrays of a step that brings n tokens of each sequence, with pages handed out in random order"""
    B, n, pasts, pages = c["B"], c["n"], _pasts(c), _pages(c)
    i32 = dict(dtype=torch.int32, device=DEV)
    total, most = sum(pages), max(pages)
    count = torch.tensor(pages, device=DEV)
    first = torch.cumsum(count, 0) - count
    col = torch.arange(most, device=DEV)
    perm = torch.randperm(total, device=DEV, generator=g)
    table = torch.where(col[None] < count[:, None], perm[(first[:, None] + col[None]).clamp(max=total - 1)], torch.zeros((), dtype=torch.long, device=DEV))
    pos0 = torch.tensor(pasts, **i32)
    return dict(ent=torch.arange(B, **i32).repeat_interleave(n), pos=(pos0[:, None] + torch.arange(n, **i32)[None]).reshape(-1).contiguous(),
                start=torch.arange(0, B * n + 1, n, **i32), slot=torch.arange(B, **i32), pos0=pos0, bt=table.to(torch.int32).contiguous()), total


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + 17) & 0x7FFFFFFF)
    rnd = lambda *s: torch.randn(s, device=DEV, generator=g)
    k = c["kind"]
    if k == "store":
        G, D, T = c["G"], c["D"], c["B"] * c["n"]
        st, total = _step(c, g)
        ty = torch.float32 if c["type"] == "f32" else torch.bfloat16
        pool = lambda: torch.zeros((total, G, BS * _groups(D) * 20), dtype=torch.uint8, device=DEV)
        return dict(case=c, st=st, k=(rnd(T, G * D) + 2.0 * rnd(G * D)).to(ty), v=rnd(T, G * D).to(ty), kpool=pool(), vpool=pool())
    if k == "attend":
        H, G, D, T = c["H"], c["G"], c["D"], c["B"] * c["n"]
        st, total = _step(c, g)
        NG = _groups(D)
        return dict(case=c, st=st, q=rnd(T, H * D), kpool=_rand_pool(total, G, NG, 1.0, g), vpool=_rand_pool(total, G, NG, 0.1, g))
    if k == "copy":
        P, n, G, D = c["pages"], c["copied"], c["G"], c["D"]
        if c["bits"] == 4:
            pools = [_rand_pool(P, G, _groups(D), 1.0, g) for _ in range(c["pools"])]
        else:
            pools = [rnd(P, BS, G, D) for _ in range(c["pools"])]
        perm = torch.randperm(P, device=DEV, generator=g)
        src, dst = perm[:n], perm[n:2 * n]
        return dict(case=c, pools=pools, src=src, dst=dst, pairs=list(zip(src.tolist(), dst.tolist())))
    R, V = c["R"], c["V"]
    lens = torch.randint(max(1, c["hist"] // 2), c["hist"] + 1, (R,), device=DEV, generator=g)
    hs = torch.zeros(R + 1, dtype=torch.int32, device=DEV)
    hs[1:] = torch.cumsum(lens, 0)
    # tokens come again, as they do in text: small ids far more often than large ones
    hist = (torch.rand(R * c["hist"], device=DEV, generator=g) ** 4 * V).to(torch.int32).clamp(max=V - 1)[:int(hs[-1])].contiguous()
    rules = torch.stack([1.0 + 0.5 * torch.rand(R, device=DEV, generator=g), 0.6 * torch.rand(R, device=DEV, generator=g), 0.4 * torch.rand(R, device=DEV, generator=g),
                         0.5 + torch.rand(R, device=DEV, generator=g)], 1).contiguous()
    s = dict(case=c, logits=3.0 * rnd(R, V), out=torch.empty((R, V), device=DEV), hist=hist, hist_start=hs, prompt=(lens // 2).to(torch.int32), rules=rules, bias=None, mask=None)
    if c["bias"]:
        ids = torch.rand((R, V), device=DEV, generator=g).topk(c["bias"], 1).indices.to(torch.int32).reshape(-1).contiguous()
        s["bias"] = (torch.arange(0, R * c["bias"] + 1, c["bias"], dtype=torch.int32, device=DEV), ids, 2.0 * rnd(R * c["bias"]))
    if c["mask"]:
        s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (R, -(-V // 32)), dtype=torch.int32, device=DEV, generator=g)
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------------------
def _padded(x, G, D):
    """[T, G * D] -> f32 [T, G, groups, 32], and which of those are values of the row"""
    P = 32 * _groups(D)
    x = x.float().reshape(-1, G, D)
    if P > D:
        x = torch.cat([x, x[..., -1:].expand(-1, -1, P - D)], -1)     # repeated: in a group that has values they change neither end
    real = (torch.arange(P, device=DEV) < D).reshape(-1, 32)
    return x.reshape(-1, G, P // 32, 32), real


def _quantised(x, G, D):
    """(steps f16, minima f16, codes) of rows, group by group"""
    x, real = _padded(x, G, D)
    x = x.clamp(-32000.0, 32000.0)
    low = x.amin(-1, keepdim=True).half()
    step = ((x.amax(-1, keepdim=True) - low.float()) * FIFTEENTH).clamp(min=0.0)
    step = ((step.view(torch.int32) + 0x1FFFF) & ~0x1FFFF).view(torch.float32)           # seven significant bits, upwards
    step = torch.where(step < 2.0 ** -18, torch.ceil(step * 2.0 ** 24) * 2.0 ** -24, step)
    inv = torch.where(step > 0, 1.0 / step, torch.zeros_like(step))
    code = torch.round((x - low.float()) * inv).clamp(0, 15).to(torch.int32)
    used = real.any(-1)[None, None, :, None]
    return torch.where(used, step, 0.0).half(), torch.where(used, low.float(), 0.0).half(), torch.where(real[None, None], code, 0)


def _slots(s):
    """page and place in the page of every token of the step"""
    st = s["st"]
    pos = st["pos"].long()
    return st["bt"].long()[st["ent"].long(), pos // BS], pos % BS


def _split(pool, NG):
    """views of a pool's bytes: codes [pages, G, rows, bytes], parameters [pages, G, rows, groups, 2]"""
    p, G = pool.shape[:2]
    codes = pool[..., :BS * NG * 16].reshape(p, G, BS, NG * 16)
    return codes, pool[..., BS * NG * 16:].contiguous().view(torch.float16).reshape(p, G, BS, NG, 2)


def _fields(word, n):
    return (word[..., None] >> (4 * torch.arange(n, device=DEV, dtype=torch.int32))) & 15


def _values(codes, par, key):
    """f32 values of rows of codes (uint8 [..., 16 NG]) and parameters (f16 [..., NG, 2])"""
    NG = par.shape[-2]
    lead = codes.shape[:-1]
    if key:
        f = _fields(codes.contiguous().view(torch.int32).reshape(*lead, 4, NG), 8).transpose(-3, -2)        # [group, part, 8]
    else:
        f = _fields(codes.contiguous().view(torch.int16).to(torch.int32).reshape(*lead, 8, NG), 4).transpose(-3, -2)
    f = f.reshape(*lead, NG, 32).float()
    return (f * par[..., :1].float() + par[..., 1:].float()).reshape(*lead, NG * 32)


def _store_plain(s):
    c = s["case"]
    G, D = c["G"], c["D"]
    NG = _groups(D)
    page, at = _slots(s)
    read = []
    for name, key in (("k", True), ("v", False)):
        step, low, code = _quantised(s[name], G, D)
        n, width = (4, 8) if key else (8, 4)
        word = (code.reshape(-1, G, NG, n, width) << (4 * torch.arange(width, device=DEV, dtype=torch.int32))).sum(-1).transpose(-2, -1)      # [part, group]
        word = (word.to(torch.int32) if key else word.to(torch.int16)).contiguous()
        pool = s[name + "pool"]
        pool[..., :BS * NG * 16].unflatten(-1, (BS, NG * 16))[page, :, at] = word.reshape(-1, G, NG * n).view(torch.uint8).reshape(-1, G, NG * 16)
        par = torch.stack([step[..., 0], low[..., 0]], -1).contiguous()
        pool[..., BS * NG * 16:].unflatten(-1, (BS, NG * 4))[page, :, at] = par.reshape(-1, G, 2 * NG).view(torch.uint8).reshape(-1, G, 4 * NG)
        codes, params = pool[..., :BS * NG * 16].unflatten(-1, (BS, NG * 16))[page, :, at], pool[..., BS * NG * 16:].unflatten(-1, (BS, NG * 4))[page, :, at]
        read.append(_values(codes, params.contiguous().view(torch.float16).reshape(-1, G, NG, 2), key)[..., :D].reshape(-1, G * D))
    return tuple(read)


def _seen(c, kpos, qpos):
    see = kpos <= qpos
    return see & (qpos - kpos < c["window"]) if c["window"] else see


def _attend_plain(s):
    c = s["case"]
    B, n, H, G, D = c["B"], c["n"], c["H"], c["G"], c["D"]
    NG, R = _groups(D), H // G
    bt, pos0 = s["st"]["bt"].long(), s["st"]["pos0"].long()
    L = bt.shape[1] * BS
    rows = []
    for name, key in (("kpool", True), ("vpool", False)):
        codes, par = _split(s[name], NG)
        x = _values(codes[bt], par[bt], key)[..., :D]                                # [B, pages, G, rows, D]
        rows.append(x.transpose(1, 2).reshape(B, G, L, D))
    q = s["q"].reshape(B, n, G, R, D).permute(0, 2, 3, 1, 4).reshape(B, G, R * n, D)
    z = (q @ rows[0].transpose(-1, -2)) * D ** -0.5
    qpos = (pos0[:, None] + torch.arange(n, device=DEV)[None]).repeat(1, R)              # [B, R * n]
    z = z.masked_fill(~_seen(c, torch.arange(L, device=DEV), qpos[..., None])[:, None], float("-inf"))
    w = torch.exp(z - z.amax(-1, keepdim=True))
    o = (w @ rows[1]) / w.sum(-1, keepdim=True)
    o = o.reshape(B, G, R, n, D).permute(0, 3, 1, 2, 4).reshape(B * n, H * D)
    return o if c["type"] == "f32" else o.bfloat16()


def _logits_plain(s):
    c = s["case"]
    R, V = c["R"], c["V"]
    row = torch.repeat_interleave(torch.arange(R, device=DEV), (s["hist_start"][1:] - s["hist_start"][:-1]).long(), output_size=s["hist"].numel())
    at = torch.arange(row.numel(), device=DEV) - s["hist_start"].long()[row]
    flat = row * V + s["hist"].long()
    seen = torch.zeros(R * V, device=DEV).index_put((flat,), torch.ones((), device=DEV))
    count = torch.zeros(R * V, device=DEV).index_put((flat,), (at >= s["prompt"].long()[row]).float(), accumulate=True)
    seen, count = seen.reshape(R, V) > 0, count.reshape(R, V)
    rep, pres, freq, temp = (s["rules"][:, i:i + 1] for i in range(4))
    x = s["logits"]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - count * freq - (count > 0).float() * pres
    if s["bias"] is not None:
        start, ids, vals = s["bias"]
        x = x.reshape(-1).index_add(0, torch.arange(R, device=DEV).repeat_interleave(c["bias"]) * V + ids.long(), vals).reshape(R, V)
    x = x / temp
    if s["mask"] is not None:
        bits = (s["mask"][..., None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        x = x.masked_fill(bits.reshape(R, -1)[:, :V] == 0, float("-inf"))
    return x


# ---- one pass ----------------------------------------------------------------------------------------------------------------------
def _handles(s):
    """what a program makes once for a layer and a step: the step's descriptor, the layer's, the output rows"""
    if "desc" not in s:
        from blazr_b200 import seqops
        c, st = s["case"], s["st"]
        T = c["B"] * c["n"]
        s["desc"] = seqops.StepDesc(st["ent"].data_ptr(), st["pos"].data_ptr(), st["start"].data_ptr(), st["slot"].data_ptr(), st["pos0"].data_ptr(), st["bt"].data_ptr(),
                                    T, c["B"], st["bt"].shape[1], BS)
        if c["kind"] == "attend":
            s["layer"] = seqops.attn_desc(c["H"], c["G"], c["D"], c["D"], c["D"] ** -0.5, gated=False, window=c["window"], kv_shared=True)
            s["out"] = torch.empty((T, c["H"] * c["D"]), dtype=torch.float32 if c["type"] == "f32" else torch.bfloat16, device=DEV)
        else:
            s["out"] = [torch.empty((T, c["G"] * c["D"]), device=DEV) for _ in range(2)]
    return s["desc"]


def run(state):
    s = state
    c = s["case"]
    k = c["kind"]
    if own:
        from blazr_b200 import seqops
        if k == "store":
            st = _handles(s)
            seqops.kv4_store(s["k"], s["v"], st, s["kpool"], s["vpool"])
            seqops.kv4_load(s["kpool"], s["vpool"], st, s["out"][0], s["out"][1])
            return tuple(s["out"])
        if k == "attend":
            st = _handles(s)
            seqops.attn_kv4(s["q"], st, s["layer"], s["kpool"], s["vpool"], s["out"])
            return s["out"]
        if k == "copy":
            seqops.copy_pages(s["pools"], s["pairs"])
            return s["pools"]
        start, ids, vals = s["bias"] if s["bias"] is not None else (None, None, None)
        seqops.process_logits(s["logits"], s["rules"], s["out"], hist=s["hist"], hist_start=s["hist_start"], hist_prompt=s["prompt"], bias_start=start, bias_ids=ids,
                              bias_vals=vals, mask=s["mask"])
        return s["out"]
    if k == "store":
        return _store_plain(s)
    if k == "attend":
        return _attend_plain(s)
    if k == "copy":
        for p in s["pools"]:
            p[s["dst"]] = p[s["src"]]
        return s["pools"]
    return _logits_plain(s)


def work(case):
    c = case
    k = c["kind"]
    if k == "store":
        rows = 2 * c["B"] * c["n"] * c["G"]
        packed = 20 * _groups(c["D"])
        return dict(bytes=rows * (c["D"] * (4 if c["type"] == "f32" else 2) + 2 * packed + 4 * c["D"]), flops=rows * c["D"] * 8)
    if k == "attend":
        n, H, G, D = c["n"], c["H"], c["G"], c["D"]
        pairs = keys = 0
        for p in _pasts(c):
            w = c["window"] or p + n
            keys += min(p + n, w + n - 1)
            pairs += sum(min(p + i + 1, w) for i in range(n))
        return dict(bytes=40 * _groups(D) * keys * G + c["B"] * n * H * D * (4 + (4 if c["type"] == "f32" else 2)), flops=4 * pairs * H * D)
    if k == "copy":
        page = c["G"] * BS * (20 * _groups(c["D"]) if c["bits"] == 4 else 4 * c["D"])
        return dict(bytes=2 * c["copied"] * c["pools"] * page, flops=0)
    R, V = c["R"], c["V"]
    return dict(bytes=R * (8 * V + 3 * c["hist"] + 8 * c["bias"] + (V // 8 if c["mask"] else 0)), flops=6 * R * V)


# ---- definitions in 64 bits ----------------------------------------------------------------------------------------------------------
def _f32(x):
    return x.float().double()          # a result that the definition rounds to 32 bits


def _exact_rows(x, G, D):
    """what rows [T, G * D] become: the definition rounds the range, the step, its reciprocal, the difference and the product to 32 bits"""
    out = []
    for g0 in range(0, D, 32):
        y = x.double().reshape(-1, G, D)[..., g0:g0 + 32].clamp(-32000, 32000)
        low = y.min(-1, keepdim=True).values.half().double()
        step = _f32(_f32(y.max(-1, keepdim=True).values - low) * FIFTEENTH).clamp(min=0)
        m, e = torch.frexp(step)
        step = torch.ldexp(torch.ceil(m * 128) / 128, e)
        step = torch.where(step < 2.0 ** -18, torch.ceil(step * 2.0 ** 24) / 2.0 ** 24, step)
        code = torch.round(_f32(_f32(y - low) * _f32(1 / step.clamp(min=2.0 ** -30)))).clamp(0, 15)
        out.append(torch.where(step > 0, code, torch.zeros_like(code)) * step + low)
    return torch.cat(out, -1).reshape(-1, G * D)


def _exact_pool(pool, table, G, D, key):
    """rows f64 [positions, G, D] that a sequence's pages stand for, bit fields taken one by one"""
    NG = _groups(D)
    b = pool[table.long()].long()                                                     # [pages, G, bytes]
    r, d = torch.arange(BS, device=DEV)[:, None], torch.arange(D, device=DEV)[None]
    g, i = d // 32, d % 32
    nibble = ((i // 8 * NG + g) * 8 + i % 8) if key else ((i // 4 * NG + g) * 4 + i % 4)
    code = (b[..., r * NG * 16 + nibble // 2] >> (4 * (nibble % 2))) & 15               # [pages, G, rows, D]
    at = BS * NG * 16 + (r * NG + g) * 4
    par = [(b[..., at + o] + 256 * b[..., at + o + 1]).to(torch.int32).to(torch.int16).view(torch.float16).double() for o in (0, 2)]
    return (code * par[0] + par[1]).permute(0, 2, 1, 3).reshape(-1, G, D)


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    k = c["kind"]
    if k == "store":
        return tuple(_exact_rows(s[n], c["G"], c["D"]) for n in ("k", "v"))
    if k == "copy":
        return None
    if k == "attend":
        H, G, D, n, pages = c["H"], c["G"], c["D"], c["n"], _pages(c)
        out = torch.zeros((c["B"] * n, H, D), dtype=torch.float64, device=DEV)
        for e, past in enumerate(_pasts(c)):
            lo = max(0, (past - c["window"] + 1) // BS) if c["window"] else 0
            tab = s["st"]["bt"][e, lo:pages[e]]
            K, V = (_exact_pool(s[p], tab, G, D, p == "kpool") for p in ("kpool", "vpool"))
            i, j = torch.arange(past, past + n, device=DEV)[:, None], lo * BS + torch.arange(K.shape[0], device=DEV)[None]
            hidden = (j > i) | (i - j >= c["window"] if c["window"] else j < 0)
            q = s["q"][e * n:(e + 1) * n].double().reshape(n, H, D)
            for h in range(H):
                z = (q[:, h] @ K[:, h * G // H].T / math.sqrt(D)).masked_fill(hidden, -math.inf)
                out[e * n:(e + 1) * n, h] = torch.softmax(z, 1) @ V[:, h * G // H]
        return out.reshape(c["B"] * n, H * D)
    x, hs = s["logits"].double(), s["hist_start"].tolist()
    for r in range(c["R"]):
        h, p = s["hist"][hs[r]:hs[r + 1]].long(), int(s["prompt"][r])
        rep, pres, freq, temp = s["rules"][r].double()
        u = torch.unique(h)
        x[r, u] = torch.where(x[r, u] > 0, x[r, u] / rep, x[r, u] * rep)
        cnt = torch.bincount(h[p:], minlength=c["V"])
        x[r] -= torch.where(cnt > 0, cnt * freq + pres, torch.zeros_like(freq))
        if s["bias"] is not None:
            at = slice(r * c["bias"], (r + 1) * c["bias"])
            x[r, s["bias"][1][at].long()] += s["bias"][2][at].double()
        x[r] /= temp
        if s["mask"] is not None:
            v = torch.arange(c["V"], device=DEV)
            x[r, (s["mask"][r].long()[v // 32] >> (v % 32)) % 2 == 0] = -math.inf
    return x
