"""Performance cases of the operators that take a queue of requests from their
prompts to their next tokens, beside the scan, the adapters and the draw.

* "int8":   a projection in 8-bit integers, a scale for each token (formed in
            the call from its largest value) and for each output channel;
* "adjust": penalties for repeated tokens, biases and grammar masks on the
            logits, before a token is drawn from them;
* "conv":   the short causal convolution with SiLU over a pool of windows,
            ragged lengths and idle rows, as the ragged scan takes them.

Sizes are those of the 8B model that the package serves (4096 hidden channels,
8192 inner ones, 18560 rows of the input projection, 10240 convolved channels,
256000 tokens) and, in the drawn cases, other head layouts and odd sizes.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

H, P, G, N, D_MODEL, D_INNER, VOCAB = 128, 64, 8, 128, 4096, 8192, 256000
IN_ROWS = 2 * D_INNER + 2 * G * N + H
LAYOUTS = ((128, 64, 8), (128, 64, 8), (80, 64, 1), (32, 128, 4), (24, 40, 3))
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one request's next token, input projection: latency and the weights' bytes
        dict(name="int8_token_b1", kind="int8", rows=1, n_in=D_MODEL, n_out=IN_ROWS, x="f16", y="f16"),
        # a full batch's next tokens, output projection
        dict(name="int8_token_b64", kind="int8", rows=64, n_in=D_INNER, n_out=D_MODEL, x="f16", y="f16"),
        # the head of a batch, logits kept in binary32
        dict(name="int8_head_b24", kind="int8", rows=24, n_in=D_MODEL, n_out=VOCAB, x="f16", y="f32"),
        # a short prompt through a small layer of odd sizes, in bfloat16
        dict(name="int8_odd", kind="int8", rows=77, n_in=1000, n_out=2041, x="bf16", y="bf16"),
        # a prompt of odd length, output projection
        dict(name="int8_prompt", kind="int8", rows=901, n_in=D_INNER, n_out=D_MODEL, x="f16", y="f16"),
        # a prefill window, input projection
        dict(name="int8_window", kind="int8", rows=2048, n_in=D_MODEL, n_out=IN_ROWS, x="f16", y="f16"),
        # one request's next token, one setting for all tokens: latency
        dict(name="adjust_b1", kind="adjust", batch=1, vocab=VOCAB, logits="f16", prompt=500, tokens=37, ragged=False,
             bias=0, masks=0),
        # a batch in which every request has settings, biases and a grammar of its own (some without)
        dict(name="adjust_b64", kind="adjust", batch=64, vocab=VOCAB, logits="f32", prompt=2048, tokens=500,
             ragged=True, bias=40, masks=48),
        # long documents, a vocabulary of odd size
        dict(name="adjust_long_b8", kind="adjust", batch=8, vocab=50003, logits="bf16", prompt=100000, tokens=4001,
             ragged=True, bias=5, masks=0),
        # decode of a full batch out of a larger pool of windows, three requests idle
        dict(name="conv_token_b64", kind="conv", batch=64, tokens=1, ragged=False, pool=80, idle=3, fresh=False,
             heads=H, dim=P, groups=G),
        # the prompts of a waiting queue, padded to the longest (an odd length)
        dict(name="conv_queue_b9", kind="conv", batch=9, tokens=901, ragged=True, pool=12, idle=0, fresh=False,
             heads=H, dim=P, groups=G),
        # one long document
        dict(name="conv_long_b1", kind="conv", batch=1, tokens=8192, ragged=False, pool=1, idle=0, fresh=True,
             heads=H, dim=P, groups=G),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ones' ranges, none of them again."""
    shapes = [{key: value for key, value in case.items() if key != "name"} for case in listed()]
    case = _draw(rng)
    while case in shapes:
        case = _draw(rng)
    return case


def _draw(rng):
    kind = rng.choice(("int8", "int8", "adjust", "conv"))
    if kind == "int8":
        n_in, n_out = rng.choice(((D_MODEL, IN_ROWS), (D_INNER, D_MODEL), (D_MODEL, D_INNER), (1000, 2041),
                                  *((_log(rng, 100, 8000), _log(rng, 100, 18000)) for _ in range(2))))
        return dict(kind=kind, rows=_log(rng, 1, 2048), n_in=n_in, n_out=n_out, x=rng.choice(("f16", "f16", "bf16")),
                    y=rng.choice(("f16", "f16", "bf16", "f32")))
    if kind == "adjust":
        vocab = _log(rng, 500, VOCAB)
        batch = _log(rng, 1, min(64, 64 * VOCAB // vocab))
        return dict(kind=kind, batch=batch, vocab=vocab, logits=rng.choice(tuple(TYPES)),
                    prompt=rng.choice((0, _log(rng, 1, 100000 // batch))), tokens=rng.choice((0, _log(rng, 1, 4000))),
                    ragged=rng.random() < 0.6, bias=rng.choice((0, 0, _log(rng, 1, 300))),
                    masks=rng.choice((0, 0, _log(rng, 1, 64))))
    heads, dim, groups = rng.choice(LAYOUTS)
    tokens = 1 if rng.random() < 0.3 else _log(rng, 2, 6000)
    batch = _log(rng, 1, min(64, max(1, 8192 // tokens)))
    return dict(kind=kind, batch=batch, tokens=tokens, ragged=rng.random() < 0.5, pool=batch + rng.randrange(4),
                idle=min(batch - 1, rng.randrange(3)), fresh=rng.random() < 0.5, heads=heads, dim=dim, groups=groups)


# ---------------------------------------------------------------- inputs
def _int8_inputs(case, gen, dev):
    rows, k, n = case["rows"], case["n_in"], case["n_out"]
    x = torch.randn(rows, k, generator=gen, device=dev)
    # a few channels far above the others, as activations have them; tokens of different sizes
    x[:, torch.randint(0, k, (max(1, k // 500),), generator=gen, device=dev)] *= 12.0
    x *= torch.rand(rows, 1, generator=gen, device=dev) * 2.0 + 0.1
    codes = torch.empty(n, k, dtype=torch.int8, device=dev)
    scale = torch.empty(n, device=dev)
    for part in range(0, n, 32768):   # the checkpoint's weights, in parts that fit beside the rest
        w = torch.randn(min(32768, n - part), k, generator=gen, device=dev) / math.sqrt(k)
        t = w.abs().amax(1, keepdim=True) / 127.0
        codes[part:part + 32768] = torch.round(w / t).to(torch.int8)
        scale[part:part + 32768] = t[:, 0]
    return dict(x=x.to(TYPES[case["x"]]), codes=codes, scale=scale, y=TYPES[case["y"]])


def _ids(gen, dev, batch, count, vocab):
    """Text's token ids: some far more often than others."""
    u = torch.rand(batch, count, generator=gen, device=dev)
    return (vocab ** u - 1.0).long().clamp(0, vocab - 1)


def _counts(case, what):
    """The ids of each row's list: all of them, or (ragged) from none to all."""
    if not case["ragged"]:
        return [case[what]] * case["batch"]
    rng = random.Random("%s %d %d" % (what, case["batch"], case[what]))
    return [case[what]] + [rng.randrange(case[what] + 1) for _ in range(case["batch"] - 1)]


def _adjust_inputs(case, gen, dev):
    b, v = case["batch"], case["vocab"]
    logits = torch.randn(b, v, generator=gen, device=dev) * 3.0

    def pick(values):
        at = torch.randint(0, len(values), (b,), generator=gen, device=dev)
        return torch.tensor(values, device=dev)[at]

    s = dict(logits=logits.to(TYPES[case["logits"]]), prompt=None, prompt_lengths=None, tokens=None, lengths=None,
             bias=None, allowed=None, allowed_rows=None)
    if case["prompt"]:
        s["prompt"] = _ids(gen, dev, b, case["prompt"], v)
    if case["tokens"]:
        s["tokens"] = _ids(gen, dev, b, case["tokens"], v)
    if case["ragged"]:
        for list_, lengths in (("prompt", "prompt_lengths"), ("tokens", "lengths")):
            if case[list_]:
                s[lengths] = torch.tensor(_counts(case, list_), dtype=torch.int32, device=dev)
        s.update(repetition=pick((1.0, 1.05, 1.2, 1.3)), presence=pick((0.0, 0.0, 0.4, 1.0)),
                 frequency=pick((0.0, 0.1, 0.5, -0.2)))
    else:
        s.update(repetition=1.1, presence=0.3, frequency=0.2)
    if case["bias"]:   # different ids in a row; the last few places are unused
        ids = torch.stack([torch.randperm(v, generator=gen, device=dev)[:case["bias"]] for _ in range(b)])
        ids = torch.nn.functional.pad(ids, (0, case["bias"] - ids.shape[1] + 3), value=-1).to(torch.int32)
        s["bias"] = (ids, torch.randn(ids.shape, generator=gen, device=dev) * 5.0)
    if case["masks"]:   # grammars that allow little or nearly everything; some rows have none
        words = -(-v // 32)
        dense = torch.rand(case["masks"], 1, 1, generator=gen, device=dev)
        bits = torch.rand(case["masks"], words, 32, generator=gen, device=dev) < dense
        weight = 2 ** torch.arange(32, device=dev)
        packed = (bits * weight).sum(-1)
        s["allowed"] = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)
        s["allowed_rows"] = torch.randint(-1, case["masks"], (b,), generator=gen, device=dev).to(torch.int32)
    return s


def _conv_inputs(case, gen, dev):
    b, length = case["batch"], case["tokens"]
    sizes = (case["heads"] * case["dim"], case["groups"] * N, case["groups"] * N)
    c = sum(sizes)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    # the projection's columns: z before them, dt behind
    rows = normal(b, length, sizes[0] + c + case["heads"]).half()
    s = dict(value=rows[..., sizes[0]:sizes[0] + c], sizes=sizes, weight=(normal(c, 4) * 0.4).half(),
             bias=(normal(c) * 0.1).half())
    # channels next to each other in memory, as the mixer keeps its window
    shape = (case["pool"], 4, c)
    window = torch.zeros(shape, device=dev) if case["fresh"] else normal(*shape)
    s["window"] = window.half().permute(0, 2, 1)
    slots = torch.randperm(case["pool"], generator=gen, device=dev)[:b].to(torch.int32)
    if case["idle"]:
        slots[torch.randperm(b, generator=gen, device=dev)[:case["idle"]]] = -1
    s["slots"] = slots
    s["lengths"] = torch.tensor(_counts(case, "tokens"), dtype=torch.int32, device=dev) if case["ragged"] else None
    return s


@torch.no_grad()
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = {"int8": _int8_inputs, "adjust": _adjust_inputs, "conv": _conv_inputs}[case["kind"]](case, gen, dev)
    s["kind"] = case["kind"]
    if own and case["kind"] == "int8":   # the handle that a server keeps for a projection's weights
        s["weight"] = _package("int8").Int8Weight(s["codes"], s["scale"])
    return s


# ---------------------------------------------------------------- the framework's calls
def _package(name):
    root = str(Path(__file__).resolve().parents[1] / "mamb2_8b_fp4_recall_sq3.25_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import importlib
    return importlib.import_module("mamba2_recall." + name)


def _run_own(s):
    if s["kind"] == "int8":
        return _package("int8").linear(s["x"], s["weight"], dtype=s["y"])
    if s["kind"] == "adjust":
        return _package("sampling").adjust(s["logits"], prompt=s["prompt"], prompt_lengths=s["prompt_lengths"],
                                           tokens=s["tokens"], lengths=s["lengths"], repetition=s["repetition"],
                                           presence=s["presence"], frequency=s["frequency"], bias=s["bias"],
                                           allowed=s["allowed"], allowed_rows=s["allowed_rows"])
    x, b, c = _package("full_state").convolve(s["value"], s["weight"], s["bias"], s["window"], s["sizes"],
                                              lengths=s["lengths"], slots=s["slots"])
    return dict(x=x, B=b, C=c, window=s["window"])


# ---------------------------------------------------------------- the plain forms
def _int8_plain(s):
    """Products over 1,024 inputs at a time: their integer sums are exact in binary32."""
    x = s["x"].float()
    top = x.abs().amax(1, keepdim=True)
    codes = torch.where(top > 0, torch.round(x * 127.0 / top), 0.0)
    out = []
    for n in range(0, s["codes"].shape[0], 32768):
        w, total = s["codes"][n:n + 32768], 0
        for k in range(0, x.shape[1], 1024):
            total = total + (codes[:, k:k + 1024] @ w[:, k:k + 1024].float().T).to(torch.int32)
        out.append((total.float() * (top / 127.0) * s["scale"][n:n + 32768]).to(s["y"]))
    return torch.cat(out, 1)


def _per_row(value, like):
    return torch.as_tensor(value, dtype=torch.float32, device=like.device).expand(like.shape[0])[:, None]


def _times(ids, lengths, like):
    """How often each token is in a row's list."""
    times = torch.zeros(like.shape, dtype=torch.int32, device=like.device)
    if ids is None:
        return times
    live = torch.ones_like(ids, dtype=torch.int32)
    if lengths is not None:
        live = (torch.arange(ids.shape[1], device=ids.device) < lengths[:, None]).to(torch.int32)
    return times.scatter_add_(1, ids.long(), live)


def _adjust_plain(s):
    l = s["logits"].float()
    count = _times(s["tokens"], s["lengths"], l)
    seen = (count > 0) | (_times(s["prompt"], s["prompt_lengths"], l) > 0)
    r = _per_row(s["repetition"], l)
    l = torch.where(seen, torch.where(l > 0, l / r, l * r), l)
    cost = _per_row(s["frequency"], l) * count.float() + _per_row(s["presence"], l)
    l = torch.where(count > 0, l - cost, l)
    if s["bias"] is not None:
        ids, values = s["bias"]
        used = ids >= 0
        l = l.scatter_add(1, ids.clamp(min=0).long(), torch.where(used, values, 0.0))
    if s["allowed"] is not None:
        rows = s["allowed_rows"]
        token = torch.arange(l.shape[1], device=l.device)
        words = s["allowed"][rows.clamp(min=0).long()][:, token // 32]
        free = (words >> (token % 32)) & 1
        l = torch.where((free == 1) | (rows < 0)[:, None], l, -math.inf)
    return l.to(s["logits"].dtype)


def _conv_plain(s):
    value = s["value"].float()
    b, length, c = value.shape
    active = s["slots"] >= 0
    count = torch.full((b,), length, device=value.device) if s["lengths"] is None else s["lengths"].long()
    count = torch.where(active, count, 0)
    slots = s["slots"].long()
    window = s["window"][slots.clamp(min=0)].transpose(1, 2)                    # [B, 4, C]
    series = torch.cat((window.float(), value), 1)                              # token t at 4 + t
    weight = s["weight"].float()
    o = sum(series[:, 1 + j:1 + j + length] * weight[:, j] for j in range(4)) + s["bias"].float()
    o = o / (1.0 + torch.exp(-o))
    live = torch.arange(length, device=value.device) < count[:, None]
    o = torch.where(live[..., None], o, 0.0).half()
    x, bm, cm = (t.contiguous() for t in torch.split(o, s["sizes"], -1))
    at = count[:, None] + torch.arange(4, device=value.device)
    last = series.gather(1, at[..., None].expand(b, 4, c)).half().transpose(1, 2)
    spare = torch.cat((s["window"], torch.zeros_like(s["window"][:1])))         # idle rows write to a spare one
    spare.index_copy_(0, torch.where(active, slots, s["window"].shape[0]), last)
    s["window"].copy_(spare[:-1])
    return dict(x=x, B=bm, C=cm, window=s["window"])


@torch.no_grad()
def run(s):
    if own:
        return _run_own(s)
    return {"int8": _int8_plain, "adjust": _adjust_plain, "conv": _conv_plain}[s["kind"]](s)


# ---------------------------------------------------------------- work
def work(case):
    if case["kind"] == "int8":
        rows, k, n = case["rows"], case["n_in"], case["n_out"]
        return dict(bytes=2 * rows * k + n * k + 4 * n + rows * n * (4 if case["y"] == "f32" else 2),
                    flops=2 * rows * k * n)
    if case["kind"] == "adjust":
        b, v = case["batch"], case["vocab"]
        size = 4 if case["logits"] == "f32" else 2
        ids = sum(_counts(case, "prompt")) + sum(_counts(case, "tokens"))
        # each logit read and written once, ids, biases, mask bits; a division, a product and two sums a logit
        return dict(bytes=2 * b * v * size + 8 * ids + 8 * b * case["bias"] + (b * v // 8 if case["masks"] else 0),
                    flops=4 * b * v)
    c = case["heads"] * case["dim"] + 2 * case["groups"] * N
    counts = _counts(case, "tokens")
    share = (case["batch"] - case["idle"]) / case["batch"]
    rows = sum(n > 0 for n in counts) * share
    # inputs read, outputs written (zeros past a row's end, too), windows read and written
    return dict(bytes=2 * c * (sum(counts) * share + case["batch"] * case["tokens"] + 8 * rows) + 10 * c,
                flops=12 * c * sum(counts) * share)


# ---------------------------------------------------------------- 64 bits
def _int8_exact(s):
    x = s["x"].double()
    top = torch.linalg.vector_norm(x, math.inf, dim=1)
    codes = torch.round(127.0 * x / torch.where(top > 0, top, 1.0)[:, None])
    out = []
    for part, scale in zip(s["codes"].split(8192), s["scale"].split(8192)):
        out.append(codes @ part.double().T * (top[:, None] / 127.0 * scale.double()))
    return torch.cat(out, 1)


def _adjust_exact(s):
    """Row by row, from the lists of ids themselves."""
    l = s["logits"].double()
    b, v = l.shape

    def values(name):
        return torch.as_tensor(s[name], dtype=torch.float32).expand(b).double().tolist()

    r, p, f = values("repetition"), values("presence"), values("frequency")
    for i in range(b):
        def list_of(ids, lengths):
            if s[ids] is None:
                return torch.zeros(0, dtype=torch.long, device=l.device)
            return s[ids][i, :None if s[lengths] is None else int(s[lengths][i])]
        new = torch.bincount(list_of("tokens", "lengths"), minlength=v).double()
        old = torch.bincount(list_of("prompt", "prompt_lengths"), minlength=v)
        at = ((new > 0) | (old > 0)).nonzero()[:, 0]
        had = l[i, at]
        l[i, at] = torch.maximum(had, had * 0) / r[i] + torch.minimum(had, had * 0) * r[i]
        l[i] -= new * f[i] + (new > 0) * p[i]
        if s["bias"] is not None:
            for token, amount in zip(s["bias"][0][i].tolist(), s["bias"][1][i].double().tolist()):
                if token >= 0:
                    l[i, token] += amount
        if s["allowed"] is not None and int(s["allowed_rows"][i]) >= 0:
            words = s["allowed"][int(s["allowed_rows"][i])].long() & 0xffffffff
            bits = (words[:, None] // (1 << torch.arange(32, device=l.device))) % 2
            l[i, bits.flatten()[:v] == 0] = -math.inf
    return l


def _conv_exact(s):
    """Row by row, the convolution over the window and the row's own tokens."""
    b, length, c = s["value"].shape
    o = torch.zeros(b, length, c, dtype=torch.float64, device=s["value"].device)
    pool = s["window"].double()
    weight, bias = s["weight"].double(), s["bias"].double()
    for i, slot in enumerate(s["slots"].tolist()):
        n = length if s["lengths"] is None else int(s["lengths"][i])
        if slot < 0 or n == 0:
            continue
        series = torch.cat((pool[slot], s["value"][i, :n].double().T), 1)      # [C, 4 + n]
        z = (series[:, 1:].unfold(1, 4, 1) * weight[:, None]).sum(-1) + bias[:, None]
        o[i, :n] = (z * torch.sigmoid(z)).T
        pool[slot] = series[:, -4:]
    x, bm, cm = torch.split(o, s["sizes"], -1)
    return dict(x=x, B=bm, C=cm, window=pool)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return {"int8": _int8_exact, "adjust": _adjust_exact, "conv": _conv_exact}[case["kind"]](s)
