"""Operators between two steps of a serving loop, as cases that can be timed and checked one by one.

  weigh    the soft-max weight that the tokens of a step (single tokens, drafts, prompt portions) give to every cached key of their sequence, added up
           per key head; keys that the step itself brought begin at zero
  evict    sequences that hold more than `keep` keys are cut back to the first ones, the most recent ones and those of largest weight between, in every
           layer and key head on their own: rows of keys and values and their weights go, in order, to the places 0 .. keep - 1 of other pages and another slot
           (a fork that goes on with fewer keys than its source)
  verify   drafted tokens against the target's probabilities, from given random numbers: how many are accepted, and the token behind them

Pages hold 16 positions, f32 [pages, 16, G, D] or in 4 bits: for every head codes of 16 rows (16 NG bytes a row, NG = 1, 2, 4 groups of 32 values), then their (s, m) pairs in f16
(4 NG bytes a row); a value is m + s * code.  Codes of a key row: 32-bit words [part c < 4][group g < NG], eight values 32 g + 8 c + i in 4-bit fields from the lowest; of a value
row 16-bit words [part r < 8][group g], four values 32 g + 4 r + i.

Row r of an entry's logits z with temperature T: w = exp((z - max z) / T), kept where z is at least the k-th largest and the kept weights of strictly larger z are below top_p of their
sum; p = w / sum.  Draft x of row i is accepted when u q(x) < p(x); q is the distribution it was drawn from, or certain.  The token behind the accepted ones comes from max(p - q, 0) of
the row that rejected, or from the last row's p: the lowest one whose cumulated weight exceeds u times their sum.

`own` chooses between the plain forms below (elementary torch operations in 32 bits, probabilities in 64: they are compared with random numbers) and the framework's calls.
"""
import math

import torch

DEV = "cuda:0"
own = False
BS = 16                     # tokens of a page: the engine's default


def listed():
    return [
        # one decoded token behind a short context: the smallest call
        dict(name="weigh_1_token", kind="weigh", B=1, n=1, last=0, past=500, ragged=False, H=32, G=8, D=64, window=0, bits=32),
        # 32 sequences decode behind contexts of 2000 to 4000 tokens
        dict(name="weigh_32_sequences", kind="weigh", B=32, n=1, last=0, past=4000, ragged=True, H=32, G=8, D=128, window=0, bits=32),
        # one sequence decodes behind a context of 128 k tokens
        dict(name="weigh_131072_keys", kind="weigh", B=1, n=1, last=0, past=131071, ragged=False, H=32, G=8, D=128, window=0, bits=32),
        # every token of a prompt of odd length counts
        dict(name="weigh_2047_tokens", kind="weigh", B=1, n=2047, last=0, past=0, ragged=False, H=32, G=8, D=128, window=0, bits=32),
        # the last 64 tokens of a long prompt's last portion choose what stays
        dict(name="weigh_last_64", kind="weigh", B=1, n=500, last=64, past=30000, ragged=False, H=32, G=8, D=64, window=0, bits=32),
        # 16 sequences with five draft tokens each, 4-bit cache
        dict(name="weigh_16x5_4bit", kind="weigh", B=16, n=5, last=0, past=1500, ragged=True, H=32, G=8, D=128, window=0, bits=4),
        # one layer of one sequence
        dict(name="evict_1_layer", kind="evict", L=1, B=1, rows=620, keep=512, first=4, recent=128, G=8, D=64, bits=32),
        # two long sequences in four layers
        dict(name="evict_2x32768", kind="evict", L=4, B=2, rows=32768, keep=16384, first=4, recent=1000, G=8, D=128, bits=32),
        # eight sequences of sixteen layers, 4-bit cache
        dict(name="evict_16_layers_4bit", kind="evict", L=16, B=8, rows=2301, keep=2048, first=4, recent=512, G=8, D=128, bits=4),
        # four drafts of one sequence that were certain (found in its own text), a 32 k vocabulary
        dict(name="verify_4_drafts", kind="verify", B=1, n=4, V=32000, probs=False, rules=False),
        # 64 sequences with four drafts each from a smaller model, a 128 k vocabulary
        dict(name="verify_64x4", kind="verify", B=64, n=4, V=128256, probs=True, rules=False),
        # the same with top_k and top_p, an odd vocabulary
        dict(name="verify_16x3_top", kind="verify", B=16, n=3, V=50257, probs=True, rules=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["weigh", "weigh", "weigh", "evict", "evict", "verify", "verify"])
    if kind == "evict":
        bits, G, D = rng.choice([4, 32]), rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128])
        L, B = rng.randint(1, 8), rng.choice([1, 1, 2, 5])
        rows = _log(rng, 40, 131072 // (L * B))
        keep = rng.randint(max(20, rows // 2), rows)
        return dict(kind=kind, L=L, B=B, rows=rows, keep=keep, first=rng.choice([0, 1, 4]), recent=rng.randint(1, keep // 2), G=G, D=D, bits=bits)
    if kind == "verify":
        return dict(kind=kind, B=_log(rng, 1, 64), n=rng.randint(0, 4), V=rng.choice([16384, 32000, 50257, 128256]), probs=rng.random() < 0.5, rules=rng.random() < 0.5)
    H, G, D = rng.choice([(32, 8, 64), (32, 8, 128), (32, 4, 128), (16, 4, 64), (16, 16, 80), (8, 1, 64), (12, 4, 96)])
    form, window, bits = rng.choice(["token", "token", "drafts", "last", "prompt"]), rng.choice([0, 0, 0, 0, 300]), rng.choice([32, 32, 4])
    if form == "token":
        B = _log(rng, 1, 64)
        return dict(kind=kind, B=B, n=1, last=0, past=_log(rng, 1, min(100000, 131072 // B)), ragged=True, H=H, G=G, D=D, window=window, bits=bits)
    if form == "drafts":
        B = _log(rng, 1, 32)
        return dict(kind=kind, B=B, n=rng.randint(2, 9), last=0, past=_log(rng, 1, 32768 // B), ragged=True, H=H, G=G, D=D, window=window, bits=bits)
    if form == "last":
        n = _log(rng, 20, 500)
        return dict(kind=kind, B=1, n=n, last=rng.choice([1, 8, 17, 32]), past=_log(rng, 100, 30000), ragged=False, H=H, G=G, D=D, window=window, bits=bits)
    n = _log(rng, 17, 2000)
    return dict(kind=kind, B=1, n=n, last=0, past=rng.choice([0, 0, _log(rng, 16, 700)]) if n < 1000 else 0, ragged=False, H=H, G=G, D=D, window=window, bits=bits)


# ---- inputs -----------------------------------------------------------------------------------------------------------------------
def _groups(D):
    return 1 if D <= 32 else 2 if D <= 64 else 4


def _spread(most, B, ragged=True):
    """B lengths: all the same, or spread evenly from half of the largest on"""
    return [most - ((i * 7919) % B * (most // 2)) // B if ragged else most for i in range(B)]


def _pool(pages, G, D, bits, mean, g):
    """pages of random rows around a mean that differs from channel to channel, as keys have it; in 4 bits random codes with steps and minima that give unit spread"""
    if bits == 32:
        return torch.randn((pages, BS, G, D), device=DEV, generator=g) + mean * torch.randn((G, D), device=DEV, generator=g)
    NG, rows = _groups(D), pages * G * BS
    codes = torch.randint(0, 256, (rows, NG * 16), dtype=torch.uint8, device=DEV, generator=g)
    step = (torch.randint(70, 128, (rows, NG), device=DEV, generator=g).float() / 512).half()
    low = (mean * torch.randn(NG, device=DEV, generator=g) - 7.5 * step.float() + 0.1 * torch.randn((rows, NG), device=DEV, generator=g)).half()
    par = torch.stack([step, low], -1).contiguous().view(torch.uint8).reshape(rows, NG * 4)
    return torch.cat([codes.reshape(-1, BS * NG * 16), par.reshape(-1, BS * NG * 4)], 1).reshape(pages, G, BS * NG * 20).contiguous()


def _tables(counts, g, extra=0):
    """int32 [B, most] block tables of sequences that hold `counts` pages, handed out in random order from sum(counts) + extra pages"""
    total, most = sum(counts), max(counts)
    count = torch.tensor(counts, device=DEV)
    first = torch.cumsum(count, 0) - count
    col = torch.arange(most, device=DEV)
    perm = torch.randperm(total + extra, device=DEV, generator=g)
    at = (first[:, None] + col[None]).clamp(max=total - 1)
    return torch.where(col[None] < count[:, None], perm[at], torch.zeros((), dtype=torch.long, device=DEV)).to(torch.int32).contiguous(), total + extra


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + 29) & 0x7FFFFFFF)
    rnd = lambda *s: torch.randn(s, device=DEV, generator=g)
    uni = lambda *s: torch.rand(s, device=DEV, generator=g)
    i32 = dict(dtype=torch.int32, device=DEV)
    k = c["kind"]
    if k == "weigh":
        B, n, H, G, D = c["B"], c["n"], c["H"], c["G"], c["D"]
        pasts = _spread(c["past"], B, c["ragged"])
        bt, total = _tables([-(-(p + n) // BS) for p in pasts], g)
        pos0 = torch.tensor(pasts, **i32)
        st = dict(ent=torch.arange(B, **i32).repeat_interleave(n), pos=(pos0[:, None] + torch.arange(n, **i32)[None]).reshape(-1).contiguous(),
                  start=torch.arange(0, B * n + 1, n, **i32), slot=torch.randperm(B + 2, device=DEV, generator=g)[:B].to(torch.int32), pos0=pos0, bt=bt)
        # weights that earlier tokens left: most keys have little
        acc = uni(B + 2, G, c["past"] + n + 5) ** 4
        return dict(case=c, st=st, q=rnd(B * n, H * D), kpool=_pool(total, G, D, c["bits"], 0.5, g), acc=acc)
    if k == "evict":
        L, B, G, D = c["L"], c["B"], c["G"], c["D"]
        rows = _spread(c["rows"], B)
        both, total = _tables([-(-r // BS) for r in rows] + [-(-min(r, c["keep"]) // BS) for r in rows], g)
        slots = torch.randperm(2 * B, device=DEV, generator=g).to(torch.int32)
        pool = lambda m: [_pool(total, G, D, c["bits"], m, g) for _ in range(L)]
        return dict(case=c, rows=torch.tensor(rows, **i32), bt=both[:B].contiguous(), to=both[B:].contiguous(), slot=slots[:B].contiguous(), to_slot=slots[B:].contiguous(),
                    kpools=pool(0.5), vpools=pool(0.1), accs=[uni(2 * B, G, c["rows"] + 3) ** 4 for _ in range(L)])
    B, n, V = c["B"], c["n"], c["V"]
    R = B * (n + 1)
    z = 3.0 * rnd(R, V)
    # one sequence in four is greedy
    temp = torch.where(torch.arange(B, device=DEV) % 4 == 3, torch.zeros((), device=DEV), 0.5 + uni(B))
    s = dict(case=c, logits=z, start=torch.arange(0, R + 1, n + 1, **i32), temp=temp, accept_u=uni(R), sample_u=uni(B), top_k=None, top_p=None, probs=None)
    if c["rules"]:
        s["top_k"] = torch.randint(0, 200, (B,), device=DEV, generator=g).clamp(min=20).to(torch.int32) * (torch.arange(B, device=DEV) % 3 != 1).to(torch.int32)
        s["top_p"] = torch.where(torch.arange(B, device=DEV) % 3 != 0, 0.5 + 0.5 * uni(B), torch.ones((), device=DEV))
    if c["probs"]:      # a smaller model's logits are near the larger one's
        heat = temp.clamp(min=0.3).repeat_interleave(n + 1)[:, None]
        zd = (z + 0.5 * rnd(R, V)) / heat
        s["probs"] = torch.softmax(zd, 1)
        s["drafts"] = (zd - torch.log(-torch.log(uni(R, V).clamp(min=1e-30)))).argmax(1).to(torch.int32)
    else:               # right more often than not
        s["drafts"] = torch.where(uni(R) < 0.7, z.argmax(1), torch.randint(0, V, (R,), device=DEV, generator=g)).to(torch.int32)
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------------------
def _split(pool, NG):
    """views of a 4-bit pool's bytes: codes [pages, G, rows, bytes], parameters [pages, G, rows, bytes]"""
    return pool[..., :BS * NG * 16].unflatten(-1, (BS, NG * 16)), pool[..., BS * NG * 16:].unflatten(-1, (BS, NG * 4))


def _key_rows(pool, bt, G, D, bits):
    """f32 keys [B, G, positions, D] of the pages of block tables"""
    B = bt.shape[0]
    if bits == 32:
        return pool[bt].permute(0, 3, 1, 2, 4).reshape(B, G, -1, D)
    NG = _groups(D)
    codes, par = _split(pool, NG)
    codes, par = codes[bt].contiguous().view(torch.int32), par[bt].contiguous().view(torch.float16).float()       # [B, pages, G, rows, 4 NG], [.., 2 NG]
    f = (codes[..., None] >> (4 * torch.arange(8, device=DEV, dtype=torch.int32))) & 15
    f = f.unflatten(-2, (4, NG)).transpose(-3, -2).flatten(-2).float()                                             # [.., NG, 32]
    par = par.unflatten(-1, (NG, 2))
    x = (f * par[..., :1] + par[..., 1:]).flatten(-2)[..., :D]
    return x.transpose(1, 2).reshape(B, G, -1, D)


def _weigh_plain(s):
    c, st = s["case"], s["st"]
    B, n, H, G, D = c["B"], c["n"], c["H"], c["G"], c["D"]
    R, m = H // G, min(c["last"] or n, n)
    K = _key_rows(s["kpool"], st["bt"].long(), G, D, c["bits"])
    L = min(K.shape[2], s["acc"].shape[2])
    q = s["q"].reshape(B, n, G, R, D)[:, n - m:].permute(0, 2, 3, 1, 4).reshape(B, G, R * m, D)
    z = (q @ K[:, :, :L].transpose(-1, -2)) * D ** -0.5
    pos0 = st["pos0"].long()
    qpos = (pos0[:, None] + torch.arange(n - m, n, device=DEV)[None]).repeat(1, R)[..., None]
    j = torch.arange(L, device=DEV)
    see = (j <= qpos) & (qpos - j < c["window"]) if c["window"] else j <= qpos
    z = z.masked_fill(~see[:, None], float("-inf"))
    w = torch.exp(z - z.amax(-1, keepdim=True))
    w = (w / w.sum(-1, keepdim=True)).sum(2)                                              # [B, G, L]
    old = s["acc"][st["slot"].long(), :, :L]
    new = torch.where((j[None] < pos0[:, None])[:, None], old + w, w)
    s["acc"][st["slot"].long(), :, :L] = torch.where((j[None] < pos0[:, None] + n)[:, None], new, old)
    return s["acc"]


def _evict_plain(s):
    c = s["case"]
    B, G, D, keep, bits = c["B"], c["G"], c["D"], c["keep"], c["bits"]
    slot, to_slot, rows = s["slot"].long(), s["to_slot"].long(), s["rows"].long()
    acc = torch.stack([a[slot] for a in s["accs"]])                                       # [L, B, G, cap]
    j, n = torch.arange(acc.shape[-1], device=DEV), rows[None, :, None, None]
    sure = (j < c["first"]) | (j >= n - c["recent"]) | (n <= keep)
    rank = torch.where(j < n, torch.where(sure, float("inf"), acc), float("-inf"))
    width = min(keep, acc.shape[-1])
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :width]
    kept = torch.sort(torch.where(kept < n, kept, acc.shape[-1]), dim=-1).values
    live = (kept < n)[0, :, 0]                                                            # [B, width]: the same for all layers and heads
    kept = torch.where(kept < n, kept, torch.full_like(kept, -1))
    e, i = live.nonzero(as_tuple=True)
    dst, g = s["to"].long()[e, i // BS], torch.arange(G, device=DEV)[None]
    for l, a in enumerate(s["accs"]):
        src = kept[l][e, :, i]                                                            # [moved, G]
        a[to_slot[e][:, None], g, i[:, None]] = a[slot[e][:, None], g, src]
        page = s["bt"].long()[e[:, None], src // BS]
        for pool in (s["kpools"][l], s["vpools"][l]):
            if bits == 32:
                pool[dst[:, None], (i % BS)[:, None], g] = pool[page, src % BS, g]
            else:
                for part in _split(pool, _groups(D)):
                    part[dst[:, None], g, (i % BS)[:, None]] = part[page, g, src % BS]
    if width < keep:
        kept = torch.cat([kept, kept.new_full((*kept.shape[:-1], keep - width), -1)], -1)
    return dict(kept=kept.to(torch.int32), accs=s["accs"], kpools=s["kpools"], vpools=s["vpools"])


def _probabilities(s):
    """f64 [R, V] of what every row may give, zero where its rules leave nothing"""
    c = s["case"]
    z, per = s["logits"], c["n"] + 1
    T = s["temp"].double().repeat_interleave(per)[:, None]
    top = z.amax(1, keepdim=True)
    w = torch.exp((z.double() - top.double()) / torch.where(T > 0, T, torch.ones_like(T)))
    if c["rules"]:
        k = s["top_k"].long().repeat_interleave(per)[:, None]
        zs = torch.sort(z, dim=1, descending=True).values
        kth = torch.where(k > 0, zs.gather(1, (k - 1).clamp(min=0, max=c["V"] - 1)), zs[:, -1:])
        w = w.masked_fill(z < kth, 0.0)
        ws = torch.exp((zs.double() - top.double()) / torch.where(T > 0, T, torch.ones_like(T))).masked_fill(zs < kth, 0.0)
        share = s["top_p"].double().repeat_interleave(per)[:, None]
        n = ((torch.cumsum(ws, 1) - ws) < share * ws.sum(1, keepdim=True)).sum(1, keepdim=True).clamp(min=1)
        w = torch.where((share < 1) & (z < zs.gather(1, n - 1)), torch.zeros_like(w), w)
    at = torch.arange(c["V"], device=DEV)[None]
    best = torch.where(z == top, at, c["V"]).amin(1, keepdim=True)
    return torch.where(T > 0, w / w.sum(1, keepdim=True), (at == best).double())


def _verify_plain(s):
    c = s["case"]
    B, n, V = c["B"], c["n"], c["V"]
    p = _probabilities(s)
    x = s["drafts"].long()
    px = p.gather(1, x[:, None])[:, 0]
    qx = s["probs"].gather(1, x[:, None])[:, 0].double() if c["probs"] else torch.ones_like(px)
    greedy = (s["temp"] <= 0).repeat_interleave(n + 1)
    fine = torch.where(greedy, px > 0, s["accept_u"].double() * qx < px).reshape(B, n + 1)[:, :n]
    accepted = torch.cumprod(fine.long(), 1).sum(1)
    row = torch.arange(B, device=DEV) * (n + 1) + accepted
    w = p[row]
    if c["probs"]:
        q = s["probs"][row].double()
    else:
        q = (torch.arange(V, device=DEV)[None] == x[row][:, None]).double()
    rest = (w - q).clamp(min=0.0)
    some = (accepted < n) & (s["temp"] > 0) & (rest.sum(1) > 0)
    cum = torch.cumsum(torch.where(some[:, None], rest, w), 1)
    nxt = (cum <= s["sample_u"].double()[:, None] * cum[:, -1:]).sum(1).clamp(max=V - 1)
    i = torch.arange(n + 1, device=DEV)[None]
    tokens = torch.where(i < accepted[:, None], x.reshape(B, n + 1), torch.where(i == accepted[:, None], nxt[:, None], -1))
    return accepted.to(torch.int32), tokens.reshape(-1).to(torch.int32)


# ---- one pass ----------------------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    c = s["case"]
    k = c["kind"]
    if own:
        from blazr_b200 import seqops
        if k == "weigh":
            if "desc" not in s:     # what a program makes once for a step and for a layer
                st = s["st"]
                s["desc"] = seqops.StepDesc(st["ent"].data_ptr(), st["pos"].data_ptr(), st["start"].data_ptr(), st["slot"].data_ptr(), st["pos0"].data_ptr(), st["bt"].data_ptr(),
                                            c["B"] * c["n"], c["B"], st["bt"].shape[1], BS)
                s["layer"] = seqops.attn_desc(c["H"], c["G"], c["D"], c["D"], c["D"] ** -0.5, gated=False, window=c["window"], kv_shared=True)
            seqops.key_weights(s["q"], s["desc"], s["layer"], s["kpool"], s["acc"], last=c["last"])
            return s["acc"]
        if k == "evict":
            kept = seqops.evict_keys(s["kpools"], s["vpools"], s["accs"], s["slot"], s["rows"], s["bt"], c["keep"], first=c["first"], recent=c["recent"], block_size=BS,
                                     to_table=s["to"], to_slots=s["to_slot"])
            return dict(kept=kept, accs=s["accs"], kpools=s["kpools"], vpools=s["vpools"])
        return seqops.verify_drafts(s["logits"], s["start"], s["drafts"], s["accept_u"], s["sample_u"], s["temp"], top_k=s["top_k"], top_p=s["top_p"], draft_probs=s["probs"])
    return _weigh_plain(s) if k == "weigh" else _evict_plain(s) if k == "evict" else _verify_plain(s)


def work(case):
    c = case
    k = c["kind"]
    row = lambda: 20 * _groups(c["D"]) if c["bits"] == 4 else 4 * c["D"]
    if k == "weigh":
        n, H, G, D = c["n"], c["H"], c["G"], c["D"]
        m = min(c["last"] or n, n)
        pairs = keys = 0
        for p in _spread(c["past"], c["B"], c["ragged"]):
            w = c["window"] or p + n
            keys += min(p + n, w + m - 1)
            pairs += sum(min(p + n - m + i + 1, w) for i in range(m))
        return dict(bytes=keys * G * (row() + 8) + 4 * c["B"] * m * H * D, flops=2 * pairs * H * D)
    if k == "evict":
        rows = _spread(c["rows"], c["B"])
        kept = sum(min(r, c["keep"]) for r in rows)
        return dict(bytes=c["L"] * c["G"] * (kept * (4 * row() + 8 + 4) + 4 * sum(rows)), flops=0)
    B, n, V = c["B"], c["n"], c["V"]
    return dict(bytes=4 * V * B * (n + 1 + (1 if c["probs"] and n else 0)), flops=4 * V * B * (n + 1))


# ---- definitions in 64 bits ----------------------------------------------------------------------------------------------------------
def _exact_keys(pool, pages, g, D, bits):
    """f64 [positions, D] of head g of a sequence's pages, bit fields taken one by one"""
    if bits == 32:
        return pool[pages.long(), :, g].double().reshape(-1, D)
    NG = _groups(D)
    b = pool[pages.long(), g].long()
    r, d = torch.arange(BS, device=DEV)[:, None], torch.arange(D, device=DEV)[None]
    field = (d % 32 // 8 * NG + d // 32) * 8 + d % 8
    code = (b[:, r * NG * 16 + field // 2] >> (4 * (field % 2))) & 15
    at = BS * NG * 16 + (r * NG + d // 32) * 4
    par = [(b[:, at + o] + 256 * b[:, at + o + 1]).to(torch.int32).to(torch.int16).view(torch.float16).double() for o in (0, 2)]
    return (code * par[0] + par[1]).reshape(-1, D)


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["kind"] == "weigh":
        H, G, D, n = c["H"], c["G"], c["D"], c["n"]
        out, m = s["acc"].double(), min(c["last"] or c["n"], c["n"])
        for e, past in enumerate(_spread(c["past"], c["B"], c["ragged"])):
            i, j = torch.arange(past + n - m, past + n, device=DEV)[:, None], torch.arange(past + n, device=DEV)[None]
            hidden = (j > i) | (i - j >= c["window"] if c["window"] else j < 0)
            q = s["q"][e * n + n - m:(e + 1) * n].double().reshape(m, H, D)
            slot = int(s["st"]["slot"][e])
            out[slot, :, past:past + n] = 0.0
            for g in range(G):
                K = _exact_keys(s["kpool"], s["st"]["bt"][e, :-(-(past + n) // BS)], g, D, c["bits"])[:past + n]
                for h in range(g * H // G, (g + 1) * H // G):
                    out[slot, g, :past + n] += torch.softmax((q[:, h] @ K.T / math.sqrt(D)).masked_fill(hidden, -math.inf), 1).sum(0)
        return out
    if c["kind"] == "evict":        # moved as they are: only the weights are computed numbers
        accs = [a.double() for a in s["accs"]]
        for a, b in zip(s["accs"], accs):
            for e, n in enumerate(s["rows"].tolist()):
                for g in range(c["G"]):
                    x = a[int(s["slot"][e]), g, :n]
                    keep = list(range(n))
                    if n > c["keep"]:
                        mid = x[c["first"]:n - c["recent"]]
                        best = torch.sort(mid, descending=True, stable=True).indices[:c["keep"] - c["first"] - c["recent"]] + c["first"]
                        keep = list(range(c["first"])) + sorted(best.tolist()) + list(range(n - c["recent"], n))
                    b[int(s["to_slot"][e]), g, :len(keep)] = x[torch.tensor(keep, device=DEV)].double()
        return dict(kept=None, accs=accs, kpools=[None] * c["L"], vpools=[None] * c["L"])
    return None                     # tokens and counts
