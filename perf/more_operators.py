"""The operators of a decoding step with 4-bit weights and edited logits: measured cases and plain forms.

  pack    fp16 weights [N][K] to 4-bit codes and back. A group of `group` neighbouring k of a row has one fp16
          scale and, in the form with `least`, its smallest value:
            with least     s = rd((max - min) / 15), l = min, code = rint((x - l) * (1 / s)) in 0..15
            without        s = rd(max |x| / 7),              code = 8 + rint(x * (1 / s)),   -7..7
          (rd: to fp16, downwards; s = 0: code 0, or 8). The value that a code stands for is code * s + l, or
          (code - 8) * s, rounded to fp16. codes uint8 [N][K/2]: of the 8 elements of each 32-bit word, element 2 i
          lies in bits 4 i and element 2 i + 1 in bits 16 + 4 i. scale, least fp16 [K/group][N].
  linear  C[b, n] = e(sum_k A[b, k] * value[n, k] + bias[n]) for B rows, e: the value itself, gelu_new, or the sum
          with a residual; rounded once.
  edit    logits [rows][V] on their way to a choice: a token t that row r's history holds is divided by the
          repetition penalty (multiplied where the logit is not positive), one that it holds c times behind the prompt
          loses frequency * c + presence; listed biases are added; a token whose mask bit is 0 becomes -inf. next is the
          largest written logit's token, the lowest of equal ones.

run() computes them in plain torch operations where `own` is false, and through the library's entry points where it is
true.
"""
import math
import os
import sys

import torch

own = False

VOCAB = 50257  # GPT-2's vocabulary
PACKED = 8192 * 8192  # weights of the largest conversion
WEIGHTS = 16384 * 8192  # weights of the largest product
LOGITS = 256 * 131072  # logits of the largest edit


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # GPT-2's QKV weight of one layer, as a program converts it when it loads a checkpoint.
        dict(name="pack_qkv", op="pack", N=2304, K=768, group=64, least=False),
        # A large generic weight with the most accurate form.
        dict(name="pack_large", op="pack", N=8192, K=8192, group=128, least=True),
        # One sequence's attention projection with the residual: the smallest product, bound by latency.
        dict(name="linear_one", op="linear", B=1, N=768, K=768, group=64, least=False, epi="resid", bias=True),
        # One token through a large layer: the weights' bytes are all there is.
        dict(name="linear_token", op="linear", B=1, N=8192, K=8192, group=128, least=True, epi="store", bias=False),
        # GPT-2's tied head for eight sequences.
        dict(name="linear_head", op="linear", B=8, N=VOCAB, K=768, group=64, least=False, epi="store", bias=False),
        # A ragged shape: nothing is a multiple of a tile.
        dict(name="linear_odd", op="linear", B=19, N=4999, K=2080, group=32, least=True, epi="gelu", bias=True),
        # The QKV projection of the benchmark's 64 sequences.
        dict(name="linear_step", op="linear", B=64, N=2304, K=768, group=64, least=False, epi="store", bias=True),
        # 64 sequences through a large layer: bytes and products cost about the same.
        dict(name="linear_batch", op="linear", B=64, N=8192, K=8192, group=64, least=False, epi="store", bias=True),
        # The widest batch and the largest weight: bound by the products.
        dict(name="linear_wide", op="linear", B=256, N=16384, K=8192, group=128, least=True, epi="gelu", bias=True),
        # One sequence in the middle of a generation, penalties and the greedy choice.
        dict(name="edit_one", op="edit", type="half", rows=1, vocab=VOCAB, history=300, biases=0, mask=False, next=True),
        # The benchmark's 64 sequences near their end, each with a grammar's mask, biases and all penalties.
        dict(name="edit_batch", op="edit", type="half", rows=64, vocab=VOCAB, history=1023, biases=16, mask=True, next=True),
        # Many rows over a large vocabulary with long histories, for a sampler that reads the logits itself.
        dict(name="edit_wide_fp32", op="edit", type="float", rows=256, vocab=131072, history=8192, biases=300, mask=True, next=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["pack", "linear", "linear", "linear", "edit", "edit"])
    group, least = rng.choice([32, 64, 128]), rng.choice([False, True])
    if op == "pack":
        K = group * _log(rng, 1, 16384 // group)
        return dict(op=op, N=_log(rng, 1, min(65536, PACKED // K)), K=K, group=group, least=least)
    if op == "linear":
        B = rng.choice([1, 1, 2, _log(rng, 1, 16), _log(rng, 17, 64), _log(rng, 65, 256)])
        K = group * _log(rng, 1, 16384 // group)
        return dict(op=op, B=B, N=_log(rng, 1, min(65536, WEIGHTS // K)), K=K, group=group, least=least, epi=rng.choice(["store", "gelu", "resid"]),
                    bias=rng.choice([False, True]))
    vocab = rng.choice([VOCAB, _log(rng, 100, 131072)])
    rows = _log(rng, 1, min(1024, LOGITS // vocab))
    return dict(op=op, type=rng.choice(["half", "float"]), rows=rows, vocab=vocab, history=_log(rng, 1, max(1, min(16384, (1 << 21) // rows))),
                biases=rng.choice([0, _log(rng, 1, 300)]) if vocab > 1000 else 0, mask=rng.choice([False, True]), next=rng.choice([False, True, True]))


# ----------------------------------------------------------------------------------------- inputs
def _weights(N, K, g):
    """Weights as trained layers have them: normal, rows of unequal size, a few large elements and a few dead rows."""
    w = torch.randn(N, K, generator=g, device="cuda", dtype=torch.float16)
    w *= (0.02 * torch.exp(0.5 * torch.randn(N, 1, generator=g, device="cuda"))).half()
    at = torch.randint(0, N * K, (max(1, N * K // 5000),), generator=g, device="cuda")
    w.view(-1)[at] *= 8
    w[torch.rand(N, generator=g, device="cuda") < 0.002] = 0
    return w


def _spread(n, lo, hi):
    """n whole numbers spread evenly over lo..hi, hi the last of them."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lens(c):
    return _spread(c["rows"], (c["history"] + 1) // 2, c["history"])


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c, "op": c["op"]}
    if c["op"] == "edit":
        rows, vocab = c["rows"], c["vocab"]
        # a language model's logits: a broad body and a few likely tokens, those of the history among them
        x = 2.0 * torch.randn(rows, vocab, generator=g, device="cuda")
        x += 4.0 * (torch.rand(rows, vocab, generator=g, device="cuda") < 2e-4) * torch.rand(rows, vocab, generator=g, device="cuda")
        u = torch.rand(rows, c["history"], generator=g, device="cuda")
        s["history"] = (vocab * u**4).to(torch.int32).clamp(max=vocab - 1)  # few tokens make up most of a text
        x.scatter_(1, s["history"][:, : max(1, c["history"] // 8)].long(), 9.0 + 0.01 * (seed % 7))
        s["logits"] = x.to(torch.float16 if c["type"] == "half" else torch.float32)
        s["length"] = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")[torch.randperm(rows, generator=g, device="cuda")].contiguous()
        s["prompt"] = (s["length"] * torch.rand(rows, generator=g, device="cuda")).to(torch.int32)
        s["repetition"] = 1.0 + 0.5 * torch.rand(rows, generator=g, device="cuda")
        s["frequency"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
        s["presence"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
        s["bias_token"] = s["bias"] = s["mask"] = None
        if c["biases"]:
            some = torch.randperm(vocab, generator=g, device="cuda")[: c["biases"]]
            move = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda")
            s["bias_token"] = ((some + move) % vocab).to(torch.int32)
            s["bias"] = 3.0 * torch.randn(rows, c["biases"], generator=g, device="cuda")
        if c["mask"]:  # a grammar allows a part of the vocabulary, in runs
            words = (vocab + 31) // 32
            keep = torch.rand(rows, words, generator=g, device="cuda") < 0.3
            bits = torch.randint(-(2**31), 2**31, (rows, words), generator=g, device="cuda")
            s["mask"] = torch.where(keep, bits, 0).to(torch.int32)
            s["mask"][:, vocab // 64] |= 1
        s["out"] = torch.empty_like(s["logits"])
        s["next"] = torch.empty(rows, dtype=torch.int32, device="cuda") if c["next"] else None
        return s
    N, K, group = c["N"], c["K"], c["group"]
    if c["op"] == "pack":
        s["w"] = _weights(N, K, g)
        s["codes"] = torch.empty(N, K // 2, dtype=torch.uint8, device="cuda")
        s["scale"] = torch.empty(K // group, N, dtype=torch.float16, device="cuda")
        s["least"] = torch.empty_like(s["scale"]) if c["least"] else None
        s["out"] = torch.empty_like(s["w"])
        return s
    s["codes"] = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    s["scale"] = (0.006 * torch.exp(0.4 * torch.randn(K // group, N, generator=g, device="cuda"))).half()
    s["least"] = (-7.5 * s["scale"].float() * (1 + 0.2 * torch.randn(K // group, N, generator=g, device="cuda"))).half() if c["least"] else None
    s["a"] = torch.randn(c["B"], K, generator=g, device="cuda", dtype=torch.float16)
    s["a"] *= torch.exp(0.5 * torch.randn(K, generator=g, device="cuda")).half()
    s["bias"] = (0.1 * torch.randn(N, generator=g, device="cuda")).half() if c["bias"] else None
    s["c0"] = torch.randn(c["B"], N, generator=g, device="cuda", dtype=torch.float16) if c["epi"] == "resid" else None
    s["out"] = torch.empty(c["B"], N, device="cuda", dtype=torch.float16)
    return s


def work(case):
    c = case
    if c["op"] == "edit":
        size, rows = 2 if c["type"] == "half" else 4, c["rows"]
        listed_bytes = 8 * c["biases"] * rows + (rows * ((c["vocab"] + 31) // 32) * 4 if c["mask"] else 0)
        return {"bytes": 2 * size * rows * c["vocab"] + 4 * sum(_lens(c)) + listed_bytes + 28 * rows, "flops": rows * c["vocab"]}
    weights = c["N"] * c["K"] // 2 + (4 if c["least"] else 2) * c["N"] * (c["K"] // c["group"])
    if c["op"] == "pack":  # read and packed, read and unpacked
        return {"bytes": 4 * c["N"] * c["K"] + 2 * weights, "flops": 6 * c["N"] * c["K"]}
    outs = c["B"] * c["N"] * (4 if c["epi"] == "resid" else 2) + (2 * c["N"] if c["bias"] else 0)
    return {"bytes": weights + 2 * c["B"] * c["K"] + outs, "flops": 2 * c["B"] * c["N"] * c["K"]}


# ------------------------------------------------------------------------------------ plain forms
PLACES = (0, 16, 4, 20, 8, 24, 12, 28)  # the bit at which each of a word's 8 elements lies


def _codes_of(codes, K):
    """The codes 0..15 [N][K] of packed ones."""
    words = codes.view(-1, K // 2).view(torch.int32)
    return torch.stack([(words >> p) & 15 for p in PLACES], -1).view(-1, K)


def _values(codes, scale, least, K, group):
    """The fp16 values that codes stand for, in 32 bits (64 before their rounding: the sum has more bits than 24)."""
    q = _codes_of(codes, K)
    sc = scale.t().repeat_interleave(group, 1).double()
    v = (q - 8) * sc if least is None else q * sc + least.t().repeat_interleave(group, 1).double()
    return v.half().float()


def _down16(x):
    """x >= 0 in 32 bits to fp16, downwards."""
    h = x.half()
    return torch.where(h.float() > x, (h.view(torch.int16) - 1).view(torch.float16), h)


def _pack(s):
    c = s["case"]
    N, K, group = c["N"], c["K"], c["group"]
    w = s["w"].float().view(N, K // group, group)
    if c["least"]:
        least = w.amin(-1)
        scale = _down16((w.amax(-1) - least) / 15.0)
        x, bottom, first, last = w - least[..., None], 0, 0.0, 15.0
    else:
        scale = _down16(w.abs().amax(-1) / 7.0)
        x, bottom, first, last = w, 8, -7.0, 7.0
    wide = scale.float()[..., None]
    inv = torch.where(wide > 0, 1.0 / wide, 0.0)
    code = ((x * inv).round().clamp(first, last) + bottom).to(torch.int32).view(N, K // 8, 8)
    words = torch.zeros(N, K // 8, dtype=torch.int32, device=w.device)
    for i, place in enumerate(PLACES):
        words |= code[..., i] << place
    s["codes"].copy_(words.view(torch.uint8))
    s["scale"].copy_(scale.t())
    if c["least"]:
        s["least"].copy_(least.t())
    return _values(s["codes"], s["scale"], s["least"], K, group).half()


def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))


def _linear(s):
    c = s["case"]
    y = s["a"].float() @ _values(s["codes"], s["scale"], s["least"], c["K"], c["group"]).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["epi"] == "gelu":
        y = _gelu(y)
    if c["epi"] == "resid":
        y = s["c0"].float() + y
    return y.half()


def _edited(s, x, wide):
    """The edited logits of x in the type `wide`."""
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    at = torch.arange(c["history"], device=x.device)
    held = at < s["length"][:, None]
    behind = held & (at >= s["prompt"][:, None])
    tokens = s["history"].long()
    seen = torch.zeros(rows, vocab, dtype=wide, device=x.device).scatter_add_(1, tokens, held.to(wide)) > 0
    count = torch.zeros(rows, vocab, dtype=wide, device=x.device).scatter_add_(1, tokens, behind.to(wide))
    rep = s["repetition"].to(wide)[:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(count > 0, x - s["frequency"].to(wide)[:, None] * count - s["presence"].to(wide)[:, None], x)
    if s["bias"] is not None:
        x = x.scatter_add(1, s["bias_token"].long(), s["bias"].to(wide))  # a token once a row
    if s["mask"] is not None:
        bits = (s["mask"][..., None] >> torch.arange(32, device=x.device)) & 1
        x = torch.where(bits.view(rows, -1)[:, :vocab] != 0, x, -math.inf)
    return x


def _first(y):
    """The first index of each row's maximum."""
    top = y.amax(-1, keepdim=True)
    at = torch.arange(y.shape[-1], device=y.device)
    return torch.where(y == top, at, y.shape[-1]).amin(-1).to(torch.int32)


def _edit(s):
    y = _edited(s, s["logits"].float(), torch.float32).to(s["logits"].dtype)
    return [y] if s["next"] is None else [y, _first(y.float())]


# -------------------------------------------------------------------------------------------- run
def _handle(s):
    """The handle that a user's program makes once: the weight's, or the edit's of a batch of sequences."""
    if "handle" not in s:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bare-metal-gpt2_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import gpt2_b200 as G
        if s["op"] == "edit":
            s["handle"] = G.LogitsEdit(G.load(), torch, s["case"]["rows"], s["case"]["vocab"], history=s["history"], length=s["length"], prompt=s["prompt"],
                                       repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"], bias_token=s["bias_token"],
                                       bias=s["bias"], mask=s["mask"])
        else:
            s["handle"] = G.W4Weight(G.load(), torch, s["codes"], s["scale"], s["least"])
            s["epi"] = {"store": G.LINEAR_STORE, "gelu": G.LINEAR_GELU, "resid": G.LINEAR_RESID}.get(s["case"].get("epi"))
    return s["handle"]


def run(state):
    s = state
    if s["op"] == "pack":
        if own:
            h = _handle(s)
            h.quantize(s["w"])
            h.dequantize(s["out"])
        out = s["out"] if own else _pack(s)
        return [out, s["scale"]] + ([] if s["least"] is None else [s["least"]])
    if s["op"] == "linear":
        if not own:
            return [_linear(s)]
        _handle(s).linear(s["out"], s["a"], s["bias"], s["epi"], s["c0"])
        return [s["out"]]
    if not own:
        return _edit(s)
    _handle(s).apply(s["out"], s["logits"], s["next"])
    return [s["out"]] if s["next"] is None else [s["out"], s["next"]]


# ------------------------------------------------------------------------------------------ exact
def _exact_pack(s):
    c = s["case"]
    N, K, group = c["N"], c["K"], c["group"]
    out, scales, leasts = torch.empty(N, K, dtype=torch.float64, device="cuda"), [], []
    for n in range(0, N, 1024):
        w = s["w"][n:n + 1024].double().unflatten(1, (-1, group))
        low = w.min(-1).values if c["least"] else -w.abs().max(-1).values
        steps = (w.max(-1).values - low) / 15 if c["least"] else -low / 7
        near = steps.half().double()
        near = torch.where(near > steps, (steps.half().view(torch.int16) - 1).view(torch.float16).double(), near)
        base = low if c["least"] else torch.zeros_like(low)
        lo, hi = (0, 15) if c["least"] else (-7, 7)
        code = torch.where(near[..., None] > 0, torch.round((w - base[..., None]) / torch.where(near > 0, near, 1.0)[..., None]), 0.0).clamp(lo, hi)
        out[n:n + 1024] = (code * near[..., None] + base[..., None]).flatten(1)
        scales.append(near)
        leasts.append(low)
    return [out, torch.cat(scales).t()] + ([torch.cat(leasts).t()] if c["least"] else [])


def _exact_linear(s):
    c = s["case"]
    out = torch.empty(c["B"], c["N"], dtype=torch.float64, device="cuda")
    a = s["a"].double()
    for n in range(0, c["N"], 2048):
        word = s["codes"][n:n + 2048].contiguous().view(torch.int16).int() & 0xFFFF  # 4 elements of one half of a word
        half = word.unflatten(1, (-1, 2))
        code = torch.empty(half.shape[0], half.shape[1], 8, dtype=torch.float64, device="cuda")
        for i in range(8):
            code[..., i] = ((half[..., i % 2] >> (4 * (i // 2))) & 15).double()
        code = code.flatten(1).unflatten(1, (-1, c["group"]))
        scale = s["scale"][:, n:n + 2048].t().double()[..., None]
        v = (code - 8) * scale if s["least"] is None else code * scale + s["least"][:, n:n + 2048].t().double()[..., None]
        out[:, n:n + 2048] = a @ v.half().double().flatten(1).t()
    if s["bias"] is not None:
        out += s["bias"].double()
    if c["epi"] == "gelu":
        out = out * 0.5 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (out + 0.044715 * out**3)))
    return [out + s["c0"].double() if c["epi"] == "resid" else out]


def _exact_edit(s):
    c = s["case"]
    y = s["logits"].double()
    for r in range(c["rows"]):
        n, p = int(s["length"][r]), int(s["prompt"][r])
        some = torch.unique(s["history"][r, :n]).long()
        x, rep = y[r, some], s["repetition"][r].double()
        y[r, some] = torch.where(x > 0, x / rep, x * rep)
        some, count = torch.unique(s["history"][r, p:n], return_counts=True)
        y[r, some.long()] -= s["frequency"][r].double() * count + s["presence"][r].double()
        if s["bias"] is not None:
            y[r, s["bias_token"][r].long()] += s["bias"][r].double()
        if s["mask"] is not None:
            token = torch.arange(c["vocab"], device="cuda")
            y[r, (s["mask"][r][token // 32] >> (token % 32)) & 1 == 0] = -math.inf
    return [y] if s["next"] is None else [y, None]


def exact(case, seed):
    s = prepare(case, seed)
    return {"pack": _exact_pack, "linear": _exact_linear, "edit": _exact_edit}[case["op"]](s)
