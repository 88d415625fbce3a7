"""Cases for timing and checking the decode operators: an 8-bit K/V cache (writing it, attending over
it) and beam search (selecting candidates, reordering the beams' states).

Cache format.  K and V of `seqs` sequences and `heads` heads are held as codes int8[seqs][heads][cap][dim]
with one exponent for each block of 16 tokens and head, int8[seqs][heads][cap / 16]: a code c of a block
with exponent e stands for c * 2^e.  Position p of a sequence lives in slot p % cap.
"""
import math
import random
import sys

import torch

own = False  # True: `run` calls the framework's kernels; False: the plain form in elementary torch operations

BLOCK = 16
EMIN = -100  # exponent of a block in which nothing but zeros was written
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one caption stream early in its utterance, the repository's own head layout: latency counts
        dict(name="attend_one", op="attend", n=1, heads=16, q_heads=16, dim=128, tokens=1, context=130, cap=768,
             window=0, dtype="f32", ragged=False),
        # every stream of the benchmark's 512, rings wrapped, the window of 751 positions that a step sees
        dict(name="attend_streams", op="attend", n=512, heads=16, q_heads=16, dim=128, tokens=1, context=1501, cap=768,
             window=751, dtype="f32", ragged=True),
        # a few long transcripts through a model with grouped heads: the split over a long axis
        dict(name="attend_long", op="attend", n=4, heads=8, q_heads=32, dim=128, tokens=1, context=65521, cap=65536,
             window=0, dtype="bf16", ragged=True),
        # two short pieces of buffered audio caught up at once, left-padded, small heads
        dict(name="prompt_small", op="attend", n=2, heads=4, q_heads=12, dim=64, tokens=37, context=301, cap=320,
             window=0, dtype="f16", ragged=True),
        # a long recording's prompt taken in large chunks
        dict(name="prompt_large", op="attend", n=4, heads=16, q_heads=16, dim=128, tokens=1024, context=4096, cap=4096,
             window=0, dtype="bf16", ragged=False),
        # one decode step's K and V of the benchmark's streams
        dict(name="append_step", op="append", n=512, heads=16, dim=128, tokens=1, context=1501, cap=768, dtype="f32"),
        # the K and V of a chunk of prompts
        dict(name="append_prompt", op="append", n=8, heads=16, dim=128, tokens=2048, context=2900, cap=4096, dtype="bf16"),
        # one utterance with four beams over the model's text vocabulary
        dict(name="select_one", op="select", batch=1, beams=4, vocab=8000, dtype="f32", eos=False),
        # a server's utterances with eight beams each
        dict(name="select_batch", op="select", batch=128, beams=8, vocab=8000, dtype="f32", eos=False),
        # a large odd vocabulary, beams that ended among the others
        dict(name="select_wide", op="select", batch=16, beams=16, vocab=65537, dtype="bf16", eos=True),
        # one layer's K/V of one utterance with four beams
        dict(name="reorder_one", op="reorder", batch=1, beams=4, segments=32, cap=751, unit=128, dtype="bf16"),
        # a server's utterances with full rings
        dict(name="reorder_batch", op="reorder", batch=32, beams=8, segments=64, cap=751, unit=128, dtype="bf16"),
    ]


def _framework():
    """The package, which lies in a folder of its own."""
    if "stt-web_b200" not in sys.path:
        sys.path.insert(0, "stt-web_b200")
    import stt_b200
    return stt_b200


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "select", "reorder"])
    if op in ("attend", "append"):
        heads, q_heads = rng.choice([(16, 16), (2, 2), (1, 8), (8, 32), (4, 12), (3, 15), (8, 64)])
        dim = rng.choice([64, 128])
        dtype = rng.choice(["f32", "bf16", "f16"])
        tokens = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 1000)])
        context = max(tokens, _log(rng, 1, 60000))
        # a ring of its own size: some wrap
        held = context if rng.random() < 0.6 else rng.randint(tokens, context)
        cap = (held + tokens + 2 * BLOCK) // BLOCK * BLOCK
        room = 1.4e9 / (heads * 2 * dim * cap)
        if op == "attend":
            room = min(room, 1.6e10 / (q_heads * tokens * cap * dim), 6e8 / (q_heads * tokens * cap))
        while room < 1:  # too large for one sequence: a shorter ring
            cap = max(BLOCK * 2, cap // 2 // BLOCK * BLOCK)
            tokens = min(tokens, cap // 2)
            context = max(context, tokens)
            room = 1.4e9 / (heads * 2 * dim * cap)
            if op == "attend":
                room = min(room, 1.6e10 / (q_heads * tokens * cap * dim), 6e8 / (q_heads * tokens * cap))
        n = _log(rng, 1, max(1, min(512, int(room))))
        case = dict(op=op, n=n, heads=heads, dim=dim, tokens=tokens, context=context, cap=cap, dtype=dtype)
        if op == "attend":
            case.update(q_heads=q_heads, window=rng.choice([0, 0, rng.randint(1, cap)]), ragged=rng.random() < 0.7)
        return case
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 24, 32])
        vocab = _log(rng, max(2, beams), 130000)
        batch = _log(rng, 1, max(1, min(256, int(1.6e7 / (beams * vocab)))))
        return dict(op=op, batch=batch, beams=beams, vocab=vocab, dtype=rng.choice(["f32", "bf16", "f16"]), eos=rng.random() < 0.4)
    beams = rng.choice([2, 3, 4, 5, 8, 12, 16])
    segments, cap, unit = _log(rng, 1, 200), _log(rng, 1, 4000), rng.choice([64, 72, 128])
    batch = _log(rng, 1, max(1, min(64, int(1.5e9 / (beams * segments * cap * unit * 4)))))
    return dict(op=op, batch=batch, beams=beams, segments=segments, cap=cap, unit=unit, dtype=rng.choice(["f32", "bf16"]))


# ------------------------------------------------------------------------------------ inputs


def _exponent(amax):
    """Smallest e >= EMIN with amax <= 127 * 2^e, for f32 amax >= 0."""
    m, ex = torch.frexp(amax)
    e = ex - 7 + (m * 128 > 127).to(ex.dtype)
    return torch.where(amax > 0, e, EMIN).clamp(min=EMIN)


def _two_to(e):
    """2^e in f32 for whole e in -126 .. 127, exact (exp2 need not be, and a tie's rounding hangs on it)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _history(seqs, heads, cap, dim, spread, gen):
    """Codes and exponents of a cache filled with N(0, spread) values, some channels larger than others."""
    dev = gen.device
    codes = torch.empty(seqs, heads, cap, dim, dtype=torch.int8, device=dev)
    exps = torch.empty(seqs, heads, cap // BLOCK, dtype=torch.int8, device=dev)
    gain = spread * (1 + 3 * (torch.rand(heads, 1, dim, generator=gen, device=dev) < 0.05).float())
    step = max(1, (1 << 27) // (heads * cap * dim))
    for i in range(0, seqs, step):
        j = min(seqs, i + step)
        x = torch.randn(j - i, heads, cap, dim, generator=gen, device=dev) * gain
        b = x.view(j - i, heads, cap // BLOCK, BLOCK, dim)
        e = _exponent(b.abs().amax((3, 4)))
        codes[i:j] = (b * _two_to(-e)[..., None, None]).round().to(torch.int8).view_as(x)
        exps[i:j] = e.to(torch.int8)
    return codes, exps


def _rows(case, gen, heads):
    """A step's [n, tokens, heads, dim] input, as a slice of wider rows where the tokens come one at a time (q, k and v of one product)."""
    n, t, d = case["n"], case["tokens"], case["dim"]
    wide = torch.randn(n, t, 2, heads, d, generator=gen, device=gen.device).to(DTYPES[case["dtype"]])
    return wide[:, :, 0] if t == 1 else wide[:, :, 0].contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    rng = random.Random(seed)
    s = dict(case)
    if case["op"] in ("attend", "append"):
        n, heads, dim, cap, t = case["n"], case["heads"], case["dim"], case["cap"], case["tokens"]
        kc, ke = _history(n, heads, cap, dim, 1.0, gen)
        vc, ve = _history(n, heads, cap, dim, 0.7, gen)
        # one piece of memory in the cache's order: the codes of K, of V, the exponents of K, of V
        mem = torch.cat([x.view(-1).view(torch.uint8) for x in (kc, vc, ke, ve)])
        a, b = kc.numel(), ke.numel()
        s["memory"] = mem
        s["kc"], s["vc"] = mem[:a].view(torch.int8).view_as(kc), mem[a:2 * a].view(torch.int8).view_as(vc)
        s["ke"], s["ve"] = mem[2 * a:2 * a + b].view(torch.int8).view_as(ke), mem[2 * a + b:].view(torch.int8).view_as(ve)
        del kc, vc, ke, ve
        # each sequence ends somewhere in the last tenth of the context where they are ragged
        last = [case["context"] - (rng.randrange(case["context"] // 10 + 1) if case.get("ragged", True) and n > 1 and i else 0) for i in range(n)]
        counts = [min(last[i], t - (rng.randrange(t // 3 + 1) if case.get("ragged", True) and t > 1 and i else 0)) for i in range(n)]
        pos = [last[i] - counts[i] for i in range(n)]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        s["pos"], s["count"] = i32(pos), i32(counts)
        order = list(range(n))
        rng.shuffle(order)  # the batch's rows in an order of their own
        s["seqs"] = i32(order)
        if own:
            s["cache"] = _framework().Kv8Cache(n, heads, dim, cap, memory=mem)
        if case["op"] == "attend":
            s["q"] = _rows(case, gen, case["q_heads"])
            # a quarter of the ragged sequences of a chunk are padded on the left
            s["start"] = i32([rng.randrange(last[i] // 3 + 1) if case["ragged"] and t > 1 and rng.random() < 0.25 else 0 for i in range(n)])
            s["scale"] = 1.0 / math.sqrt(dim)
            s["out"] = torch.zeros(n, t, case["q_heads"], dim, dtype=DTYPES[case["dtype"]], device=dev)
        else:
            s["k"] = _rows(case, gen, heads)
            s["v"] = _rows(case, gen, heads).mul_(0.7)
            # what is read back: the tokens of the blocks that the call touches, up to the last new one
            first = [p // BLOCK * BLOCK for p in pos]
            s["from"], s["many"] = i32(first), i32([p + c - f for p, c, f in zip(pos, counts, first)])
            s["out_k"] = torch.zeros(n, t + BLOCK - 1, heads, dim, dtype=DTYPES[case["dtype"]], device=dev)
            s["out_v"] = torch.zeros_like(s["out_k"])
    elif case["op"] == "select":
        rows, vocab = case["batch"] * case["beams"], case["vocab"]
        x = torch.randn(rows, vocab, generator=gen, device=dev) * 3
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["scores"] = (-20 * torch.rand(case["batch"], case["beams"], generator=gen, device=dev)).float()
        s["done"] = (torch.rand(case["batch"], case["beams"], generator=gen, device=dev) < 0.3).to(torch.uint8) if case["eos"] else None
        s["eos_id"] = rng.randrange(vocab) if case["eos"] else -1
        if own:
            s["beam"] = _framework().BeamSelector(case["batch"], case["beams"], case["vocab"])
            shape = (case["batch"], case["beams"])
            s["next"] = [torch.empty(shape, dtype=d, device=dev) for d in (torch.float32, torch.int32, torch.int32, torch.uint8)]
    else:
        batch, beams = case["batch"], case["beams"]
        s["states"] = torch.randn(batch * beams, case["segments"], case["cap"], case["unit"], generator=gen, device=dev,
                                  dtype=torch.float32).to(DTYPES[case["dtype"]])
        s["parents"] = torch.tensor([[rng.randrange(beams) for _ in range(beams)] for _ in range(batch)], dtype=torch.int32, device=dev)
        held = [rng.randint((case["cap"] + 1) // 2, case["cap"]) if i else case["cap"] for i in range(batch)]
        s["held"] = torch.tensor([h for h in held for _ in range(beams)], dtype=torch.int32, device=dev)
    return s


# ------------------------------------------------------------------------------------ the plain forms


def _values(codes, exps, seqs):
    """The cache's values in f32, the sequences in the batch's order."""
    c, e = codes[seqs].float(), _two_to(exps[seqs])
    return (c.view(*e.shape, BLOCK, c.shape[-1]) * e[..., None, None]).view(c.shape)


def _attend(s):
    seqs, pos, count = s["seqs"].long(), s["pos"].long(), s["count"].long()
    n, t, heads, group, cap = s["n"], s["tokens"], s["heads"], s["q_heads"] // s["heads"], s["cap"]
    dev = seqs.device
    end = (pos + count + BLOCK - 1) // BLOCK * BLOCK  # the ring holds the positions end - cap .. end - 1
    slot = torch.arange(cap, device=dev)
    p = end[:, None] - cap + (slot[None] - (end[:, None] - cap)) % cap  # [n, cap] position in each slot
    here = pos[:, None] + torch.arange(t, device=dev)  # [n, t]
    low = s["start"].long()[:, None].clamp(min=0).expand_as(here)
    if s["window"]:
        low = torch.maximum(low, here + 1 - s["window"])
    seen = (p[:, None] >= low[..., None]) & (p[:, None] <= here[..., None])  # [n, t, cap]
    q = s["q"].float().view(n, t, heads, group, -1).permute(0, 2, 3, 1, 4).reshape(n, heads, group * t, -1)
    scores = torch.matmul(q * s["scale"], _values(s["kc"], s["ke"], seqs).transpose(2, 3)).view(n, heads, group, t, cap)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(n, heads, group * t, cap), _values(s["vc"], s["ve"], seqs)).view(n, heads, group, t, -1)
    out = torch.where(total > 0, out / total.clamp(min=1e-38), torch.zeros_like(out))
    out = out.permute(0, 3, 1, 2, 4).reshape(n, t, heads * group, -1)
    live = torch.arange(t, device=dev) < count[:, None]
    s["out"].copy_(torch.where(live[..., None, None], out.to(s["out"].dtype), s["out"]))
    return s["out"]


def _write(codes, exps, x, s):
    """Appends x [n, tokens, heads, dim] to one half of the cache."""
    seqs, pos, count = s["seqs"].long(), s["pos"].long(), s["count"].long()
    n, t, heads, blocks = s["n"], s["tokens"], s["heads"], s["cap"] // BLOCK
    nb = (t + 2 * BLOCK - 2) // BLOCK  # blocks that t tokens can touch
    dev = seqs.device
    first = pos // BLOCK
    p = (first[:, None, None] + torch.arange(nb, device=dev)[:, None]) * BLOCK + torch.arange(BLOCK, device=dev)  # [n, nb, 16]
    token = p - pos[:, None, None]
    new = (token >= 0) & (token < count[:, None, None])
    old = token < 0
    rows = x.float()[torch.arange(n, device=dev)[:, None, None], token.clamp(0, t - 1)]  # [n, nb, 16, heads, dim]
    rows = torch.where(new[..., None, None], rows, torch.zeros_like(rows)).permute(0, 3, 1, 2, 4)  # [n, heads, nb, 16, dim]
    at = (first[:, None] + torch.arange(nb, device=dev)) % blocks  # [n, nb]
    h = torch.arange(heads, device=dev)
    where = (seqs[:, None, None], h[None, :, None], at[:, None, :])
    cb, was = codes.view(-1, heads, blocks, BLOCK, codes.shape[-1]), exps[where].int()
    base = torch.where(old.any(-1)[:, None], was, EMIN)
    e = torch.maximum(base, _exponent(rows.abs().amax((3, 4))))
    scaled = (rows * _two_to(-e)[..., None, None]).round()
    kept = cb[where].float()
    moved = (kept * _two_to((was - e).clamp(min=-126))[..., None, None]).round()
    got = torch.where(new[:, None, :, :, None], scaled, torch.where(old[:, None, :, :, None], moved, kept))
    touched = new.any(-1)[:, None].expand(n, heads, nb)
    # blocks past the last new token keep what they hold; they are written back as they were read
    i, j, k = (w.expand(n, heads, nb)[touched] for w in where)
    cb[i, j, k] = got[touched].to(torch.int8)
    exps[i, j, k] = e[touched].to(torch.int8)


def _read(codes, exps, out, s):
    seqs, first, many = s["seqs"].long(), s["from"].long(), s["many"].long()
    m = torch.arange(out.shape[1], device=seqs.device)
    slot = (first[:, None] + m) % s["cap"]
    at = (seqs[:, None, None], torch.arange(s["heads"], device=seqs.device)[None, None], slot[:, :, None])
    v = codes[at].float() * _two_to(exps[at[0], at[1], at[2] // BLOCK])[..., None]
    out.copy_(torch.where((m < many[:, None])[..., None, None], v.to(out.dtype), out))
    return out


def _select(s):
    batch, beams, vocab = s["batch"], s["beams"], s["vocab"]
    x = s["logits"].double()  # in 64 bits: the order of near candidates of two beams hangs on it
    top = x.amax(1, keepdim=True)
    logp = (x - top) - torch.log(torch.exp(x - top).sum(1, keepdim=True))
    total = (logp.view(batch, beams, vocab) + s["scores"].double()[..., None])
    if s["done"] is not None:
        ended = s["done"].bool()[..., None]
        at_eos = (torch.arange(vocab, device=x.device) == s["eos_id"])
        total = torch.where(ended, torch.where(at_eos, s["scores"].double()[..., None], torch.full_like(total, -math.inf)), total)
    best, where = torch.sort(total.view(batch, beams * vocab), dim=1, descending=True, stable=True)
    best, where = best[:, :beams], where[:, :beams]
    parents, tokens = (where // vocab).int(), (where % vocab).int()
    done = tokens == s["eos_id"]
    if s["done"] is not None:
        done = done | torch.gather(s["done"].bool(), 1, parents.long())
    return [best.float(), parents, tokens, done.to(torch.uint8)]


def _reorder(s):
    beams = s["beams"]
    rows = torch.arange(s["batch"], device=s["parents"].device)[:, None] * beams + s["parents"].long()
    took = s["states"][rows.view(-1)]
    live = torch.arange(s["cap"], device=took.device) < s["held"][:, None]
    s["states"].copy_(torch.where(live[:, None, :, None], took, s["states"]))
    return s["states"]


def run(state):
    s = state
    op = s["op"]
    if not own:
        if op == "attend":
            return _attend(s)
        if op == "append":
            _write(s["kc"], s["ke"], s["k"], s)
            _write(s["vc"], s["ve"], s["v"], s)
            return [_read(s["kc"], s["ke"], s["out_k"], s), _read(s["vc"], s["ve"], s["out_v"], s)]
        return _select(s) if op == "select" else _reorder(s)
    stream = torch.cuda.current_stream().cuda_stream
    if op == "attend":
        s["cache"].attention(s["q"], s["out"], s["pos"], count=s["count"], seqs=s["seqs"], start=s["start"],
                             window=s["window"], scale=s["scale"], stream=stream)
        return s["out"]
    if op == "append":
        s["cache"].append(s["k"], s["v"], s["pos"], count=s["count"], seqs=s["seqs"], stream=stream)
        s["cache"].read(s["out_k"], s["out_v"], s["from"], count=s["many"], seqs=s["seqs"], stream=stream)
        return [s["out_k"], s["out_v"]]
    if op == "select":
        scores, parents, tokens, done = s["next"]
        s["beam"].select(s["logits"], s["scores"], scores, parents, tokens, done=s["done"], next_done=done,
                         eos=s["eos_id"], stream=stream)
        return [scores, parents, tokens, done]
    _framework().beam_reorder(s["states"], s["parents"], held=s["held"], stream=stream)
    return s["states"]


# ------------------------------------------------------------------------------------ the work


def _seen(case):
    """Keys that a sequence's queries see, for each of its tokens, the first sequence's as an example."""
    keys = 0
    for p in range(case["context"] - case["tokens"], case["context"]):
        end = -(-case["context"] // BLOCK) * BLOCK
        low = max(0, end - case["cap"], p + 1 - case["window"] if case["window"] else 0)
        keys += max(0, p + 1 - low)
    return keys


def work(case):
    if case["op"] in ("attend", "append"):
        n, t, dim, heads, size = case["n"], case["tokens"], case["dim"], case["heads"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "attend":
        held = min(case["context"], case["cap"], case["window"] + t - 1 if case["window"] else case["context"])
        return {"bytes": n * (2 * heads * held * (dim + 1 / BLOCK) + 2 * t * case["q_heads"] * dim * size),
                "flops": 4.0 * n * case["q_heads"] * dim * _seen(case)}
    if case["op"] == "append":
        rows = n * t * heads * dim
        # K and V in, their codes out; the codes of the touched tokens back in, their values out
        return {"bytes": 2 * rows * (size + 1) + 2 * n * heads * dim * (t + (BLOCK - 1) / 2) * (1 + size), "flops": 4.0 * rows}
    if case["op"] == "select":
        rows = case["batch"] * case["beams"]
        live = 0.7 if case["eos"] else 1.0  # the logits of beams that ended need not be read
        return {"bytes": live * rows * case["vocab"] * (4 if case["dtype"] == "f32" else 2) + rows * 17, "flops": live * 3.0 * rows * case["vocab"]}
    b = case["beams"]
    row = case["segments"] * case["cap"] * (0.75 if case["batch"] > 1 else 1.0) * case["unit"] * (4 if case["dtype"] == "f32" else 2)
    # each beam that changes is written once, each beam that another one takes is read once
    return {"bytes": case["batch"] * row * ((b - 1) + b * (1 - (1 - 1 / b) ** (b - 1))), "flops": 0}


# ------------------------------------------------------------------------------------ in 64 bits


def _power(e):
    """2^e in f64 for whole e in -128 .. 127, from Python's own powers."""
    return torch.tensor([2.0 ** k for k in range(-128, 128)], dtype=torch.float64, device=e.device)[e.long() + 128]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "append":
        return [_exact_append(s["kc"], s["ke"], s["k"], s["out_k"], s), _exact_append(s["vc"], s["ve"], s["v"], s["out_v"], s)]
    if case["op"] == "select":
        x = s["logits"].double()
        logp = x - torch.logsumexp(x, 1, keepdim=True)
        total = logp.view(s["batch"], s["beams"], -1) + s["scores"].double()[..., None]
        if s["done"] is not None:
            for b, k in s["done"].nonzero().tolist():
                total[b, k] = -math.inf
                total[b, k, s["eos_id"]] = s["scores"][b, k].double()
        return [total.view(s["batch"], -1).topk(s["beams"], dim=1).values, None, None, None]
    states = s["states"].double()
    got = states.clone()
    for g, row in enumerate(s["parents"].tolist()):
        for b, parent in enumerate(row):
            i = g * s["beams"] + b
            m = int(s["held"][i])
            got[i, :, :m] = states[g * s["beams"] + parent, :, :m]
    return got


def _exact_attend(s):
    """One sequence at a time: its positions in order, each query's softmax over the ones that it sees."""
    group = s["q_heads"] // s["heads"]
    out = s["out"].double()
    pos, count, start, seqs = (s[k].tolist() for k in ("pos", "count", "start", "seqs"))
    for i in range(s["n"]):
        total = pos[i] + count[i]
        held = torch.arange(max(0, -(-total // BLOCK) * BLOCK - s["cap"]), total, device=out.device)
        slot = held % s["cap"]
        k, v = (c[seqs[i]][:, slot].double() * _power(e[seqs[i]][:, slot // BLOCK])[..., None]
                for c, e in ((s["kc"], s["ke"]), (s["vc"], s["ve"])))
        q = s["q"][i, :count[i]].double()  # [c, q_heads, dim]
        at = pos[i] + torch.arange(count[i], device=out.device)
        low = torch.full_like(at, start[i]) if not s["window"] else torch.clamp(at + 1 - s["window"], min=start[i])
        hidden = (held[None] < low[:, None]) | (held[None] > at[:, None])
        logits = torch.einsum("tghd,gkd->ghtk", q.view(count[i], s["heads"], group, -1), k) * s["scale"]
        logits.masked_fill_(hidden, -math.inf)
        p = torch.nan_to_num(torch.softmax(logits, -1), nan=0.0)
        out[i, :count[i]] = torch.einsum("ghtk,gkd->tghd", p, v).reshape(count[i], s["q_heads"], -1)
    return out


def _exact_append(codes, exps, x, out, s):
    """Block by block: the exponent that the largest new value needs, or the block's own where it holds older tokens and theirs is larger."""
    out = out.double()
    pos, count, seqs = (s[k].tolist() for k in ("pos", "count", "seqs"))
    if s["n"] * (s["tokens"] / BLOCK + 2) > 30000:
        return None
    for i in range(s["n"]):
        c, e = codes[seqs[i]], exps[seqs[i]]
        first = pos[i] // BLOCK * BLOCK
        for b in range(first, pos[i] + count[i], BLOCK):
            lo, hi = max(b, pos[i]), min(b + BLOCK, pos[i] + count[i])
            slot = b % s["cap"]
            new = x[i, lo - pos[i]:hi - pos[i]].double()  # [new, heads, dim]
            need = torch.ceil(torch.log2(new.abs().amax((0, 2)).clamp(min=1e-300) / 127)).clamp(min=EMIN)
            if lo > b:
                need = torch.maximum(need, e[:, slot // BLOCK].double())
                was = c[:, slot:slot + lo - b].double() * _power(e[:, slot // BLOCK])[:, None, None]
                new = torch.cat([was.transpose(0, 1), new])
            step = _power(need)[None, :, None]
            out[i, b - first:hi - first] = torch.round(new / step) * step
    return out
