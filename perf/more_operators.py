"""Performance cases of the latent attention operators: rotary positions, the
paged latent cache's append and decode, and the expanded prefill with its
backward pass.

Each case is one pass through one operator as a training or serving program
makes it.  Heads and head sizes are the benchmark's (16 and 32 heads; 32, 64
and 128) with a rotary part of half a head beside them; a latent of four heads'
width serves all heads.

A case is a dict of plain values:
  op       rope | append | decode | prefill | prefill_backward
  dtype    of the activations, the cache and the gradients ("bf16" or "f32")
  rope:    tokens, heads, dim, rot (the last rot channels are rotated),
           interleaved, scaling ("none", "linear" or "by_parts"), start (first position)
  append:  lengths (the sequences' lengths after the call, comma-separated),
           news (the new tokens of each), latent, rot, page, norm (whether the
           latent is normalised on the way)
  decode:  lengths, steps (new positions of every sequence), heads, latent,
           rot, page
  prefill, prefill_backward:
    lengths (queries of each sequence), prior (keys of each before its first
    query), heads, nope, rot, vdim, causal, packed (else all lengths are alike
    and the batch is dense)
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
THETA, FACTOR, TRAINED = 10000.0, 8.0, 4096


def _rope(dtype, tokens, heads, dim, rot, *, interleaved=False, scaling="none", start=0):
    return dict(op="rope", dtype=dtype, tokens=tokens, heads=heads, dim=dim, rot=rot, interleaved=interleaved,
                scaling=scaling, start=start)


def _append(dtype, lengths, news, *, latent=512, rot=64, page=64, norm=True):
    return dict(op="append", dtype=dtype, lengths=lengths, news=news, latent=latent, rot=rot, page=page, norm=norm)


def _decode(dtype, lengths, *, steps=1, heads=16, latent=512, rot=64, page=64):
    return dict(op="decode", dtype=dtype, lengths=lengths, steps=steps, heads=heads, latent=latent, rot=rot, page=page)


def _prefill(op, dtype, lengths, *, prior="", heads=32, nope=128, rot=64, vdim=128, causal=True, packed=True):
    return dict(op=op, dtype=dtype, lengths=lengths, prior=prior, heads=heads, nope=nope, rot=rot, vdim=vdim,
                causal=causal, packed=packed)


def _join(values):
    return ",".join(str(int(v)) for v in values)


def listed():
    # contexts of a serving batch, in no order
    ragged = _join(2048 + (i * 1009) % 4096 for i in range(64))
    named = {
        # one decode step's queries of a small batch: all latency
        "rope_small": _rope("bf16", 8, 32, 192, 64, start=700),
        # a training batch's queries, pairs of neighbours, positions far behind the trained length
        "rope_batch": _rope("bf16", 2 * 4096, 32, 192, 64, interleaved=True, scaling="by_parts", start=100_000),
        # one decode step's new tokens
        "append_small": _append("bf16", "900,17,1,4096,333,64,65,2047", "1,1,1,1,1,1,1,1"),
        # prompts entering the cache, one of them continuing another call's
        "append_prompts": _append("bf16", "4096,1187,9000,1,2048", "4096,1187,3001,1,2048"),
        # one request's decode step: all latency
        "decode_small": _decode("bf16", "517"),
        # a serving batch's decode step
        "decode_batch": _decode("bf16", ragged),
        # two long contexts, verified four positions at a time
        "decode_long": _decode("bf16", "131072,100001", steps=4, heads=32),
        # a short prompt of a small model
        "prefill_small": _prefill("prefill", "bf16", "64", heads=2, nope=32, rot=16, vdim=32, packed=False),
        # a prompt batch of the benchmark's lengths
        "prefill_batch": _prefill("prefill", "bf16", "4096,4096", packed=False),
        # prompts packed without padding, some continuing behind cached keys, in full precision
        "prefill_fp32": _prefill("prefill", "f32", "513,1,190,1003", prior="0,700,129,0", heads=8, nope=64, rot=32,
                                 vdim=64),
        # a training step of the same shape
        "backward_batch": _prefill("prefill_backward", "bf16", "4096,4096", packed=False),
        # documents packed without padding, in full precision
        "backward_fp32": _prefill("prefill_backward", "f32", "300,77,512,1,190", heads=8, nope=64, rot=32, vdim=64),
    }
    return [dict(name=n, **c) for n, c in named.items()]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _parts(rng, total, n):
    cuts = sorted(rng.randint(0, total) for _ in range(n - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    """One more case of the listed ones' ranges; none costs more than the largest listed."""
    op = rng.choice(["rope", "append", "decode", "decode", "prefill", "prefill", "prefill_backward",
                     "prefill_backward"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "rope":
        rot = rng.choice([16, 32, 64, 64, 128, 2 * rng.randint(1, 64)])
        dim = rot + rng.choice([0, 32, 64, 128, 128, rng.randint(0, 128)])
        heads = rng.choice([1, 2, 8, 20, 20, rng.randint(1, 40)])
        return _rope(dtype, _log_int(rng, 1, 50_000_000 // (heads * dim)), heads, dim, rot,
                     interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "by_parts"]),
                     start=_log_int(rng, 1, 200_000))
    if op in ("append", "decode"):
        latent, rot = rng.choice([(512, 64), (512, 64), (256, 32), (128, 16), (512, 0),
                                  (rng.randint(8, 512), 2 * rng.randint(1, 32))])
        page = rng.choice([16, 64, 64, 128, rng.randint(1, 200)])
        n = _log_int(rng, 1, 64)
        if op == "append":
            news = _parts(rng, _log_int(rng, n, 10_000), n)
            lens = [x + rng.choice([0, 0, _log_int(rng, 1, 2000)]) for x in news]
            return _append(dtype, _join(lens), _join(news), latent=latent, rot=rot, page=page, norm=rng.random() < 0.7)
        heads, steps = rng.choice([8, 16, 16, 32, 64, 128, rng.randint(1, 24)]), rng.choice([1, 1, 1, 2, 4, 7])
        # rows of the cache x rows of queries
        most = min(260_000, (4_000_000 if dtype == "f32" else 30_000_000) // (heads * steps))
        total = _log_int(rng, min(n * 16, most), most)
        return _decode(dtype, _join(max(steps, x) for x in _parts(rng, total, n)), steps=steps, heads=heads, latent=latent,
                       rot=rot, page=page)
    nope, rot, vdim = rng.choice([(128, 64, 128), (128, 64, 128), (64, 32, 64), (32, 16, 32), (128, 0, 128), (64, 64, 128),
                                  (rng.randint(8, 128), 2 * rng.randint(0, 32), rng.randint(8, 128))])
    heads = rng.choice([1, 2, 8, 20, 40, rng.randint(1, 20)])
    causal = rng.random() < 0.8
    most = 0.6e8 if dtype == "f32" else 2.5e8  # twice that with prior keys, in pairs x heads
    tokens = _log_int(rng, 1, int(min(16384, math.sqrt(most / heads))))
    if rng.random() < 0.4:
        b = _log_int(rng, 1, 8)
        return _prefill(op, dtype, _join([max(1, tokens // b)] * b), heads=heads, nope=nope, rot=rot, vdim=vdim,
                        causal=causal, packed=False)
    n = rng.randint(1, min(12, tokens))
    lens = _parts(rng, tokens, n)
    prior = "" if rng.random() < 0.6 else _join(rng.choice([0, _log_int(rng, 1, max(1, tokens // n))]) for _ in lens)
    return _prefill(op, dtype, _join(lens), prior=prior, heads=heads, nope=nope, rot=rot, vdim=vdim, causal=causal)


def _ints(text):
    return [int(x) for x in text.split(",")] if text else []


def _pages(lengths, page, gen):
    """A page table with the sequences' pages scattered over a pool of a few pages more."""
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=gen)[:sum(need)].tolist()
    width = max(max(need), 1)
    table, at = torch.zeros(len(need), width, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, pool


def _starts(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


def _scale(case):
    """The softmax scale: by the width of a head's query before absorption."""
    return 1.0 / math.sqrt(case["nope"] + case["rot"] if "nope" in case else case["latent"] // 4 + case["rot"])


def _inputs(case, seed):
    """The tensors of the call, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(dt)

    if case["op"] == "rope":
        s = {"x": normal(case["tokens"], case["heads"], case["dim"])}
        at = torch.arange(case["tokens"], device="cuda") % 4096 + case["start"]
        return {**s, "positions": at.to(torch.int32)}
    if case["op"] in ("append", "decode"):
        lens, D = _ints(case["lengths"]), case["latent"] + case["rot"]
        table, pool = _pages(lens, case["page"], host)
        s = {"table": table.cuda(), "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda"),
             "cache": normal(pool, case["page"], D)}
        if case["op"] == "append":
            news = _ints(case["news"])
            s["cu"] = _starts(news).cuda()
            # latent and rotary key side by side, as one projection gives them
            s["both"] = normal(sum(news), D, std=2.0)
            s["norm"] = torch.randn(case["latent"], generator=gen, device="cuda") * 0.1 + 1.0
            return s
        # logits of a spread of one to two
        s["q"] = normal(len(lens), case["steps"], case["heads"], D, std=0.8)
        return s
    H, dn, dr, dv = case["heads"], case["nope"], case["rot"], case["vdim"]
    lens = _ints(case["lengths"])
    prior = _ints(case["prior"]) or [0] * len(lens)
    keys = [a + b for a, b in zip(lens, prior)]
    lead, klead = (sum(lens),), (sum(keys),)
    if not case["packed"]:
        lead = klead = (len(lens), lens[0])
    s = {"q": normal(*lead, H, dn + dr, std=1.3)}
    kv = normal(*klead, H, dn + dv)  # one projection of the latents
    s["k"], s["v"] = kv[..., :dn], kv[..., dn:]
    if dr:
        s["k_rope"] = normal(*klead, dr)
    if case["packed"]:
        s["cu"] = _starts(lens).cuda()
        if any(prior):
            s["cu_k"] = _starts(keys).cuda()
    if case["op"] == "prefill_backward":
        # a loss's gradient, a mean over the batch: far below 1
        s["do"] = normal(*lead, H, dv, std=1e-3)
    return s


def prepare(case, seed):
    s = {"case": dict(case), **_inputs(case, seed)}
    rot = case["rot"]
    if case["op"] in ("rope", "append") and rot:
        s["freq"], s["magnitude"] = _frequencies(rot, case.get("scaling", "none"))
    if case["op"] == "prefill_backward":
        # what the forward pass kept: its output and the logarithms of its sums
        o, lse = _forward(s, case)
        s["o"], s["lse"] = o, lse
    return s


def run(state):
    s, case = state, state["case"]
    if not own:
        return _PLAIN[case["op"]](s, case)
    import rhizome_amd

    if case["op"] == "rope":
        return rhizome_amd.rope(s["x"], s["positions"], s["freq"], offset=case["dim"] - case["rot"],
                                interleaved=case["interleaved"], magnitude=s["magnitude"])
    if case["op"] == "append":
        both, c = s["both"], case["latent"]
        return rhizome_amd.latent_append(both[:, :c], both[:, c:] if case["rot"] else None, s["cache"], s["table"],
                                         s["lengths"], cu_seqlens=s["cu"], frequencies=s.get("freq"),
                                         norm_scale=s["norm"] if case["norm"] else None)
    if case["op"] == "decode":
        return rhizome_amd.latent_decode(s["q"], s["cache"], s["table"], s["lengths"], d_c=case["latent"],
                                         scale=_scale(case))
    args = dict(scale=_scale(case), causal=case["causal"], cu_seqlens=s.get("cu"), cu_seqlens_k=s.get("cu_k"))
    if case["op"] == "prefill":
        return rhizome_amd.latent_prefill(s["q"], s["k"], s["v"], s.get("k_rope"), **args)
    out = rhizome_amd.latent_prefill_backward(s["q"], s["k"], s["v"], s.get("k_rope"), s["o"], s["lse"], s["do"], **args)
    return out if case["rot"] else out[:3]


# ------------------------------------------------------------- plain forms
def _frequencies(rot, scaling):
    """Turns per position of every pair, in 64 bits, and the rotated values' magnitude."""
    f = torch.tensor([THETA ** (-2.0 * i / rot) / (2 * math.pi) for i in range(rot // 2)], dtype=torch.float64,
                     device="cuda")
    if scaling == "linear":
        return f / FACTOR, 1.0
    if scaling == "by_parts":
        keep = ((TRAINED * f - 1.0) / 31.0).clamp(0.0, 1.0)
        return f * (keep + (1.0 - keep) / FACTOR), 0.1 * math.log(FACTOR) + 1.0
    return f, 1.0


def _rotate(x, positions, freq, magnitude, interleaved):
    """x [tokens, heads, rot] in 32 bits, the angles in 64."""
    turns = positions.double()[:, None] * freq
    angle = (turns - torch.floor(turns)) * (2 * math.pi)
    cos, sin = (torch.cos(angle) * magnitude).float()[:, None], (torch.sin(angle) * magnitude).float()[:, None]
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _plain_rope(s, case):
    x, rot = s["x"], case["rot"]
    y = x.clone()
    y[..., -rot:] = _rotate(x[..., -rot:].float(), s["positions"], s["freq"], s["magnitude"],
                            case["interleaved"]).to(x.dtype)
    return y


def _rows(lengths, news, page, table):
    """Row of the cache and position of every new token, the last `news` of each sequence."""
    dev = table.device
    news, lengths = torch.tensor(news, device=dev), torch.tensor(lengths, device=dev)
    seq = torch.repeat_interleave(torch.arange(len(news), device=dev), news)
    start = torch.cumsum(news, 0) - news
    pos = torch.arange(int(news.sum()), device=dev) - start[seq] + (lengths - news)[seq]
    return table[seq, pos // page].long() * page + pos % page, pos


def _plain_append(s, case):
    c = case["latent"]
    both, cache = s["both"], s["cache"]
    rows, pos = _rows(_ints(case["lengths"]), _ints(case["news"]), case["page"], s["table"])
    x = both[:, :c].float()
    if case["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * s["norm"]
    new = x
    if case["rot"]:
        new = torch.cat((x, _rotate(both[:, None, c:].float(), pos, s["freq"], 1.0, False)[:, 0]), -1)
    cache.view(-1, cache.shape[-1])[rows] = new.to(cache.dtype)
    return cache


def _softmax(x, seen):
    """Softmax over the places that are seen and the logarithm of its sum; zeros and -inf where none is."""
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total), (torch.log(total) + top)[..., 0]


def _decode_in(s, case, dtype):
    """Sequence by sequence: its pages gathered, the products and the softmax between them."""
    n, c = case["steps"], case["latent"]
    page = case["page"]
    cache = s["cache"].view(-1, s["cache"].shape[-1])
    out, sums = [], []
    for i, length in enumerate(_ints(case["lengths"])):
        at = torch.arange(length, device=cache.device)
        keys = cache[s["table"][i, at // page].long() * page + at % page].to(dtype)
        q = s["q"][i].to(dtype)
        seen = at[None, None] <= (length - n + torch.arange(n, device=cache.device))[:, None, None]
        p, lse = _softmax((q.flatten(0, 1) @ keys.mT).view(n, case["heads"], length) * _scale(case), seen)
        out.append((p.flatten(0, 1) @ keys[:, :c]).view(n, case["heads"], c))
        sums.append(lse)
    return torch.stack(out), torch.stack(sums)


def _plain_decode(s, case):
    o, lse = _decode_in(s, case, torch.float32)
    return o.to(s["q"].dtype), lse


def _sequences(s, case):
    """Of every sequence: its first query, its queries, its first key and its keys."""
    lens = _ints(case["lengths"])
    prior = _ints(case["prior"]) or [0] * len(lens)
    q0 = k0 = 0
    for n, m in zip(lens, prior):
        yield q0, n, k0, n + m
        q0, k0 = q0 + n, k0 + n + m


def _heads_first(x, first, count, dtype):
    """[H, count, d] of a sequence of a dense or packed tensor."""
    return x.reshape(-1, *x.shape[-2:])[first:first + count].transpose(0, 1).to(dtype).contiguous()


def _keys(s, case, first, count, dtype):
    k = _heads_first(s["k"], first, count, dtype)
    if not case["rot"]:
        return k
    r = s["k_rope"].reshape(-1, case["rot"])[first:first + count].to(dtype)
    return torch.cat((k, r.expand(case["heads"], -1, -1)), -1)


def _seen(case, n, m, device):
    """Whether query i of n sees key j of m: the last query sees all of them."""
    if not case["causal"]:
        return torch.ones(n, m, dtype=torch.bool, device=device)
    return torch.arange(m, device=device) <= torch.arange(n, device=device)[:, None] + (m - n)


def _forward(s, case, dtype=torch.float32, rounded=True):
    q = s["q"]
    H, dv = case["heads"], case["vdim"]
    o = torch.zeros(q.shape[:-1].numel() // H, H, dv, dtype=q.dtype if rounded else dtype, device=q.device)
    lse = torch.empty(o.shape[:-1], dtype=dtype, device=q.device)
    for q0, n, k0, m in _sequences(s, case):
        if n == 0:
            continue
        qs, ks = _heads_first(q, q0, n, dtype), _keys(s, case, k0, m, dtype)
        p, l = _softmax(qs @ ks.mT * _scale(case), _seen(case, n, m, q.device))
        o[q0:q0 + n] = (p @ _heads_first(s["v"], k0, m, dtype)).transpose(0, 1)
        lse[q0:q0 + n] = l.T
    return o.reshape(*q.shape[:-1], dv), lse.reshape(q.shape[:-1])


def _plain_backward(s, case):
    q, H, dn, dr = s["q"], case["heads"], case["nope"], case["rot"]
    dt, scale = q.dtype, _scale(case)
    dq = torch.zeros(q.shape[:-1].numel() // H, H, dn + dr, dtype=dt, device=q.device)
    tokens = s["k"].shape[:-2].numel()
    dk, dv = (torch.zeros(tokens, H, d, dtype=dt, device=q.device) for d in (dn, case["vdim"]))
    drope = torch.zeros(tokens, dr, dtype=dt, device=q.device)
    lse_all = s["lse"].reshape(-1, H)
    for q0, n, k0, m in _sequences(s, case):
        if n == 0:
            continue
        f = torch.float32
        qs, ks, vs = _heads_first(q, q0, n, f), _keys(s, case, k0, m, f), _heads_first(s["v"], k0, m, f)
        do, o = _heads_first(s["do"], q0, n, f), _heads_first(s["o"], q0, n, f)
        seen = _seen(case, n, m, q.device)
        p = torch.where(seen, torch.exp(qs @ ks.mT * scale - lse_all[q0:q0 + n].T[..., None]), 0.0)
        dv[k0:k0 + m] = (p.mT @ do).transpose(0, 1).to(dt)
        ds = p * (do @ vs.mT - (do * o).sum(-1, keepdim=True)) * scale
        dq[q0:q0 + n] = (ds @ ks).transpose(0, 1).to(dt)
        d = ds.mT @ qs
        dk[k0:k0 + m] = d[..., :dn].transpose(0, 1).to(dt)
        drope[k0:k0 + m] = d[..., dn:].sum(0).to(dt)
    out = (dq.reshape(q.shape), dk.reshape(s["k"].shape), dv.reshape(s["v"].shape))
    return (*out, drope.reshape(s["k_rope"].shape)) if dr else out


_PLAIN = {"rope": _plain_rope, "append": _plain_append, "decode": _plain_decode, "prefill": _forward,
          "prefill_backward": _plain_backward}


# ------------------------------------------------------------------- exact
def _exact_turn(x, positions, rot, scaling, interleaved):
    """The rotation as a product of complex numbers in 64 bits."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=x.device)
    f = torch.exp(-math.log(THETA) * 2.0 * i / rot)
    size = 1.0
    if scaling == "linear":
        f = f / FACTOR
    elif scaling == "by_parts":
        share = ((TRAINED * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f, size = (1.0 - share) * f / FACTOR + share * f, 0.1 * math.log(FACTOR) + 1.0
    turn = torch.polar(torch.full((), size, dtype=torch.float64, device=x.device), positions.double()[:, None, None] * f)
    x = x.double()
    if interleaved:
        return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
    z = torch.complex(*(t.contiguous() for t in x.chunk(2, -1))) * turn
    return torch.cat((z.real, z.imag), -1)


def _exact_append(s, case):
    c, page = case["latent"], case["page"]
    cache, at = s["cache"].double(), 0
    for i, (length, n) in enumerate(zip(_ints(case["lengths"]), _ints(case["news"]))):
        x = s["both"][at:at + n, :c].double()
        at += n
        if case["norm"]:
            x = x / ((x ** 2).sum(-1, keepdim=True) / c + 1e-6).sqrt() * s["norm"].double()
        pos = torch.arange(length - n, length, device=cache.device)
        if case["rot"]:
            r = _exact_turn(s["both"][at - n:at, None, c:], pos, case["rot"], "none", False)
            x = torch.cat((x, r[:, 0]), -1)
        cache[s["table"][i].long()[pos // page], pos % page] = x
    return cache


def _exact_decode(s, case):
    n, c, page, lens = case["steps"], case["latent"], case["page"], _ints(case["lengths"])
    o = torch.empty(len(lens), n, case["heads"], c, dtype=torch.float64, device="cuda")
    lse = torch.empty(len(lens), n, case["heads"], dtype=torch.float64, device="cuda")
    for i, length in enumerate(lens):
        used = -(-length // page)
        keys = s["cache"][s["table"][i, :used].long()].flatten(0, 1)[:length].double()
        for j in range(n):
            see = length - n + j + 1
            if see <= 0:
                o[i, j], lse[i, j] = 0.0, -math.inf
                continue
            z = s["q"][i, j].double() @ keys[:see].mT * _scale(case)
            lse[i, j] = torch.logsumexp(z, -1)
            o[i, j] = torch.exp(z - lse[i, j][:, None]) @ keys[:see, :c]
    return o, lse


def _exact_prefill(s, case):
    """Head by head, with torch's own derivative of the formula where gradients are wanted."""
    H, dn, dr, dv = case["heads"], case["nope"], case["rot"], case["vdim"]
    back = case["op"] == "prefill_backward"
    q, k, v = (s[n].double().reshape(-1, H, s[n].shape[-1]) for n in ("q", "k", "v"))
    r = s["k_rope"].double().reshape(-1, dr) if dr else k.new_zeros(k.shape[0], 0)
    if back:
        d = [torch.zeros_like(t) for t in (q, k, v, r)]
        do = s["do"].double().reshape(-1, H, dv)
    o, lse = q.new_zeros(q.shape[0], H, dv), q.new_full((q.shape[0], H), -math.inf)
    q0 = k0 = 0
    lens = _ints(case["lengths"])
    for i, n in enumerate(lens):
        m = n + (_ints(case["prior"])[i] if case["prior"] else 0)
        for h in range(H if n else 0):
            leaves = [q[q0:q0 + n, h], k[k0:k0 + m, h], v[k0:k0 + m, h], r[k0:k0 + m]]
            if back:
                leaves = [t.detach().requires_grad_(True) for t in leaves]
            z = (leaves[0][:, :dn] @ leaves[1].mT + leaves[0][:, dn:] @ leaves[3].mT) * _scale(case)
            if case["causal"]:
                hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
                z = z.masked_fill(hidden, -math.inf)
            p = torch.softmax(z, -1)
            if back:
                got = torch.autograd.grad((p @ leaves[2] * do[q0:q0 + n, h]).sum(), leaves, allow_unused=True)
                d[0][q0:q0 + n, h], d[1][k0:k0 + m, h], d[2][k0:k0 + m, h] = got[:3]
                if dr:
                    d[3][k0:k0 + m] += got[3]
            else:
                o[q0:q0 + n, h], lse[q0:q0 + n, h] = p @ leaves[2], torch.logsumexp(z, -1)
        q0, k0 = q0 + n, k0 + m
    if back:
        names = ("q", "k", "v", "k_rope") if dr else ("q", "k", "v")
        return tuple(t.reshape(s[n].shape) for t, n in zip(d, names))
    return o.reshape(*s["q"].shape[:-1], dv), lse.reshape(s["q"].shape[:-1])


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rope":
        x, rot = s["x"], case["rot"]
        y = x.double()
        y[..., -rot:] = _exact_turn(x[..., -rot:], s["positions"], rot, case["scaling"], case["interleaved"])
        return y
    if case["op"] == "append":
        return _exact_append(s, case)
    if case["op"] == "decode":
        return _exact_decode(s, case)
    return _exact_prefill(s, case)


def work(case):
    """Bytes: every input and output once, of the cache the rows that are read
    or written.  Flops of the attention: two for every product's term over the
    pairs of query and key that see each other (the backward pass has five
    products, the logits' among them); of the others a few per value."""
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2.0 * n * case["dim"] * e + 4.0 * case["tokens"] + 4.0 * case["rot"],
                "flops": 3.0 * n * case["rot"]}
    if case["op"] == "append":
        n, D = sum(_ints(case["news"])), case["latent"] + case["rot"]
        return {"bytes": 2.0 * n * D * e + 4.0 * case["latent"], "flops": 5.0 * n * D}
    if case["op"] == "decode":
        lens, n, H, c = _ints(case["lengths"]), case["steps"], case["heads"], case["latent"]
        D = c + case["rot"]
        pairs = sum(max(0, x - n + 1 + j) for x in lens for j in range(n))
        rows = len(lens) * n * H
        return {"bytes": float(e) * (sum(lens) * D + rows * (D + c)) + 4.0 * rows, "flops": 2.0 * pairs * H * (D + c)}
    H, dq, dn, dr, dv = case["heads"], case["nope"] + case["rot"], case["nope"], case["rot"], case["vdim"]
    pairs, nq, nk = 0, 0, 0
    for _, n, _, m in _sequences(None, case):
        pairs += n * (m - n) + n * (n + 1) // 2 if case["causal"] else n * m
        nq, nk = nq + n, nk + m
    values = nq * H * (dq + dv) + nk * (H * (dn + dv) + dr)  # q, o, k, v and the shared key
    if case["op"] == "prefill":
        return {"bytes": float(e) * values + 4.0 * nq * H, "flops": 2.0 * pairs * H * (dq + dv)}
    grads = nq * H * dq + nk * (H * (dn + dv) + dr)
    return {"bytes": float(e) * (values + nq * H * dv + grads) + 4.0 * nq * H,
            "flops": 2.0 * pairs * H * (3 * dq + 2 * dv)}
