"""Attention over packed sequences, its bucketed position bias, and attention over a shared prefix: cases, plain forms and
64-bit results.

Where `own` is false, `run` computes the operators in plain float32 torch operations; where it is true it calls
`packed_attention` and `shared_prefix_attention` as a program does. Lengths are part of a case (comma-separated texts, one
number a sequence), so the work of a case follows from it alone; every input value comes from the seed.

With nq queries and nk keys in a sequence the last query stands at the last key: query i has position i + nk - nq, a causal
call sees keys up to that position, and the bias goes by key position minus query position.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one generated token for four short requests: the smallest call, where launches and host work count
        dict(name="tokens_small", kind="packed", lens="1,1,1,1", keys="129,1,77,300", H=8, Hk=2, D=64, dtype="bf16",
             causal=True, train=False, pad=0, buckets=0),
        # single tokens against long histories of very different lengths: bandwidth, and one sequence that is half of it
        dict(name="tokens_long", kind="packed", lens="1,1,1,1,1,1,1,1",
             keys="32760,4097,75600,1209,16384,20011,513,9000", H=40, Hk=8, D=128, dtype="fp16", causal=True,
             train=False, pad=0, buckets=0),
        # a batch of whole prompts, grouped heads, packed end to end with some rows of padding behind them
        dict(name="prompts", kind="packed", lens="4096,37,2011,1,777,6000", keys="", H=32, Hk=8, D=128, dtype="bf16",
             causal=True, train=False, pad=22, buckets=0),
        # pieces of prompts appended to what is there already (more keys than queries), beside a single token
        dict(name="prompts_append", kind="packed", lens="256,512,31,1", keys="9000,512,4111,2600", H=24, Hk=24, D=128,
             dtype="fp16", causal=True, train=False, pad=0, buckets=0),
        # one long prompt
        dict(name="prompt_long", kind="packed", lens="32760", keys="", H=24, Hk=8, D=128, dtype="bf16", causal=True,
             train=False, pad=0, buckets=0),
        # a training step over packed causal sequences, three query heads to a key head
        dict(name="prompts_train", kind="packed", lens="4096,1000,3,2049,6553,1", keys="", H=24, Hk=8, D=128,
             dtype="bf16", causal=True, train=True, pad=12, buckets=0),
        # a training step over packed clips of different sizes (17 x 30 x 27, 9 x 30 x 44 and 16 x 16 x 16 tokens): every
        # token sees its whole clip
        dict(name="clips_train", kind="packed", lens="13770,11880,4096", keys="", H=12, Hk=12, D=128, dtype="bf16",
             causal=False, train=True, pad=0, buckets=0),
        # a prompt encoder with bucketed position bias: inference of padded-free prompts
        dict(name="bias_encode", kind="packed", lens="512,226,77,300", keys="", H=64, Hk=64, D=64, dtype="fp16",
             causal=False, train=False, pad=0, buckets=32),
        # its training step, gradient of the bucket weights among the outputs
        dict(name="bias_train", kind="packed", lens="512,77,256,512,33,400,512,1", keys="", H=24, Hk=24, D=64,
             dtype="bf16", causal=False, train=True, pad=0, buckets=32),
        # three samples of one short prompt, a token each
        dict(name="shared_small", kind="shared", n=1, P=500, S=256, lens="40,1,200", H=8, Hk=8, D=64, dtype="fp16"),
        # a token for each of 48 samples of one long prompt
        dict(name="shared_tokens", kind="shared", n=1, P=16000, S=1024, H=32, Hk=8, D=128, dtype="bf16",
             lens=",".join(str(1 + 21 * i % 1024) for i in range(48))),
        # sixteen tokens at once (drafted ones to be verified) for each of 16 samples, behind a video-long prefix
        dict(name="shared_extend", kind="shared", n=16, P=32760, S=4096, H=40, Hk=8, D=128, dtype="bf16",
             lens="16,4096,700,33,2048,100,64,1999,17,513,3000,257,1024,129,4000,31"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        if work(case)["flops"] <= 2e12:
            return case


def _draw(rng):
    kind = rng.choice(["tokens", "prompts", "prompts", "train", "train", "bias", "bias", "shared", "shared"])
    dtype, D = rng.choice(["bf16", "fp16"]), rng.choice([64, 128, 128])
    Hk = rng.choice([1, 2, 3, 5, 8])
    H = Hk * rng.choice([1, 1, 2, 3, 4, 5, 8])
    if kind == "shared":
        S, n, B = _log(rng, 64, 4000), rng.choice([1, 1, 1, 2, 5, 16]), _log(rng, 1, 64)
        lens = ",".join(str(min(S, _log(rng, n, 4000))) for _ in range(B))
        return dict(kind="shared", n=n, P=_log(rng, 30, 40000), S=max(S, n), lens=lens, H=H, Hk=Hk, D=D, dtype=dtype)
    case = dict(kind="packed", H=H, Hk=Hk, D=D, dtype=dtype, keys="", causal=True, train=False, pad=0, buckets=0)
    if kind == "tokens":
        B = _log(rng, 1, 32)
        return dict(case, lens=",".join(["1"] * B), keys=",".join(str(_log(rng, 1, 40000)) for _ in range(B)))
    if kind == "bias":
        G = rng.choice([1, 1, 2])
        lens = [_log(rng, 16, 1500)] + [_log(rng, 1, 1500) for _ in range(_log(rng, 1, 12) - 1)]
        return dict(case, lens=",".join(map(str, lens)), H=Hk * G, buckets=32, causal=rng.random() < 0.3,
                    train=rng.random() < 0.6)
    lens = [_log(rng, 1, 9000) for _ in range(_log(rng, 1, 10))]
    if kind == "train":     # (sequences of one token alone have no gradient but that of v)
        lens[0] = max(lens[0], 16)
    case.update(lens=",".join(map(str, lens)), causal=rng.random() < 0.7, train=kind == "train",
                pad=rng.choice([0, 0, 1, 50]))
    if kind == "prompts" and rng.random() < 0.4:
        case["keys"] = ",".join(str(n + _log(rng, 1, 9000)) for n in lens)
    return case


# ------------------------------------------------------------------------------------------------ inputs
MAX_DISTANCE = 128


def _numbers(text):
    return [int(x) for x in text.split(",")]


def _lengths(case):
    lens = _numbers(case["lens"])
    return lens, _numbers(case["keys"]) if case["keys"] else lens


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _inputs(case, seed):
    """The tensors of a case by name."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, H, Hk, D = DTYPES[case["dtype"]], case["H"], case["Hk"], case["D"]
    normal = lambda *shape, std=1.0: (std * torch.randn(*shape, device="cuda", generator=g)).to(dt)
    if case["kind"] == "shared":
        lens = _numbers(case["lens"])
        B, n, P, S = len(lens), case["n"], case["P"], case["S"]
        return dict(q=normal(B, n, H, D, std=1.5), kp=normal(P, Hk, D), vp=normal(P, Hk, D), k=normal(B, S, Hk, D),
                    v=normal(B, S, Hk, D))
    lq, lk = _lengths(case)
    Tq, Tk = sum(lq) + case["pad"], sum(lk) + case["pad"]
    t = dict(q=normal(Tq, H, D, std=1.5), k=normal(Tk, Hk, D), v=normal(Tk, Hk, D))
    if case["train"]:
        t["dout"] = normal(Tq, H, D)
    if case["buckets"]:
        t["bias"] = torch.randn(case["buckets"], H, device="cuda", generator=g)
    return t


def _bucket(d, buckets, bidirectional):
    """The bucket of key position minus query position d: half of the (direction's) buckets one to a distance, the others
    spaced evenly in the logarithm up to MAX_DISTANCE, the last one for everything from there on. Each border is decided in
    whole numbers: distance a is in step s or beyond where (a / exact)^(n - exact) >= (MAX_DISTANCE / exact)^s."""
    n, first = (buckets // 2, buckets // 2 if d > 0 else 0) if bidirectional else (buckets, 0)
    a = abs(d) if bidirectional else max(-d, 0)
    exact = n // 2
    if a < exact:
        return first + a
    s, m = 0, n - exact
    while s + 1 < m and a ** m * exact ** (s + 1) >= MAX_DISTANCE ** (s + 1) * exact ** m:
        s += 1
    return first + exact + s


def prepare(case, seed):
    t = _inputs(case, seed)
    state = dict(case=case, **t)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    if case["kind"] == "shared":
        return dict(state, lens=ints(_numbers(case["lens"])))
    lq, lk = _lengths(case)
    state.update(cu_q=ints(_starts(lq)), cu_k=ints(_starts(lk)))
    if case["buckets"]:
        both = not case["causal"]
        if own:
            from self_trainable_or_free_attn_amd.packed import relative_buckets
            state["table"] = relative_buckets(case["buckets"], MAX_DISTANCE, bidirectional=both, device="cuda")
        else:
            state["table"] = ints([_bucket(d, case["buckets"], both) for d in range(-MAX_DISTANCE, MAX_DISTANCE + 1)])
    if case["train"] and own:
        for name in ("q", "k", "v", "bias"):
            if name in state:
                state[name].requires_grad_()
    return state


# ------------------------------------------------------------------------------------------------ passes
def run(state):
    case = state["case"]
    if not own:
        return _plain_shared(state) if case["kind"] == "shared" else _plain_packed(state)
    from self_trainable_or_free_attn_amd.packed import packed_attention, shared_prefix_attention
    if case["kind"] == "shared":
        return shared_prefix_attention(state["q"], state["kp"], state["vp"], state["k"], state["v"], state["lens"],
                                       return_lse=True)
    out = packed_attention(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"], causal=case["causal"],
                           bias=state.get("bias"), buckets=state.get("table"), return_lse=not case["train"])
    if not case["train"]:
        return out
    leaves = [state[n] for n in ("q", "k", "v", "bias") if n in state]
    return (out, *torch.autograd.grad(out, leaves, state["dout"]))


MOST_SCORES = 1 << 29


def _blocks(Hk, G, n, m):
    """(kv heads, query rows) blocks whose scores stay under MOST_SCORES values."""
    heads = max(1, min(Hk, MOST_SCORES // max(1, G * n * m)))
    rows = n if heads > 1 else max(1, min(n, MOST_SCORES // max(1, G * m)))
    return [(h, min(h + heads, Hk), r, min(r + rows, n)) for h in range(0, Hk, heads) for r in range(0, n, rows)]


def _softmax(s, seen):
    """Rows of exp(s - lse) over the seen columns, and lse; zeros and -inf where a row sees none."""
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total), (top + torch.log(total))[..., 0]


def _plain_packed(state):
    case, train = state["case"], state["case"]["train"]
    q, k, v = (state[n].float() for n in "qkv")
    H, Hk, D = case["H"], case["Hk"], case["D"]
    G, scale, buckets = H // Hk, 1 / math.sqrt(D), case["buckets"]
    lq, lk = _lengths(case)
    out = torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, device="cuda")
    if train:
        dout = state["dout"].float()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dw = torch.zeros(buckets, H, device="cuda", dtype=torch.float64)
    group = lambda x, a, b, h0, h1: x[a:b].unflatten(1, (Hk, G))[:, h0:h1].permute(1, 2, 0, 3)   # [h, G, n, D]
    heads = lambda x, a, b, h0, h1: x[a:b, h0:h1].permute(1, 0, 2)[:, None]                     # [h, 1, n, D]
    for qa, n, ka, m in zip(_starts(lq), lq, _starts(lk), lk):
        if n == 0 or m == 0:
            continue
        j = torch.arange(m, device="cuda")[None]
        for h0, h1, r0, r1 in _blocks(Hk, G, n, m):
            pos = torch.arange(r0, r1, device="cuda")[:, None] + (m - n)
            seen = j <= pos if case["causal"] else torch.ones_like(j <= pos)
            qs, ks, vs = group(q, qa + r0, qa + r1, h0, h1), heads(k, ka, ka + m, h0, h1), heads(v, ka, ka + m, h0, h1)
            s = (qs @ ks.transpose(-1, -2)) * scale
            if buckets:
                at = state["table"].long()[(j - pos).clamp(-MAX_DISTANCE, MAX_DISTANCE) + MAX_DISTANCE]
                s = s + state["bias"][:, h0 * G:h1 * G].t()[:, at].unflatten(0, (-1, G))
            p, row_lse = _softmax(s, seen)
            group(out, qa + r0, qa + r1, h0, h1)[:] = p @ vs
            lse[qa + r0:qa + r1, h0 * G:h1 * G] = row_lse.flatten(0, 1).t()
            if not train:
                continue
            do = group(dout, qa + r0, qa + r1, h0, h1)
            heads(dv, ka, ka + m, h0, h1)[:] += (p.transpose(-1, -2) @ do).sum(1, keepdim=True)
            dp = do @ vs.transpose(-1, -2)
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            group(dq, qa + r0, qa + r1, h0, h1)[:] = (ds @ ks) * scale
            heads(dk, ka, ka + m, h0, h1)[:] += (ds.transpose(-1, -2) @ qs).sum(1, keepdim=True) * scale
            if buckets:
                for i in range(buckets):
                    dw[i, h0 * G:h1 * G] += (ds * (at == i)).flatten(0, 1).sum((-1, -2), dtype=torch.float64)
    dt = DTYPES[case["dtype"]]
    if not train:
        return out.to(dt), lse
    grads = (dq.to(dt), dk.to(dt), dv.to(dt)) + ((dw.float(),) if buckets else ())
    return (out.to(dt), *grads)


def _plain_shared(state):
    case = state["case"]
    H, Hk, D, n, P = (case[x] for x in ("H", "Hk", "D", "n", "P"))
    q, kp, vp = (state[x].float() for x in ("q", "kp", "vp"))
    out = torch.zeros_like(q)
    lse = torch.empty(q.shape[:3], device="cuda")
    for b, m in enumerate(_numbers(case["lens"])):
        ks = torch.cat([kp, state["k"][b, :m].float()]).permute(1, 0, 2)[:, None]
        vs = torch.cat([vp, state["v"][b, :m].float()]).permute(1, 0, 2)[:, None]
        qs = q[b].unflatten(1, (Hk, H // Hk)).permute(1, 2, 0, 3)
        j = torch.arange(P + m, device="cuda")[None]
        last = m - n + torch.arange(n, device="cuda")[:, None]
        p, row_lse = _softmax((qs @ ks.transpose(-1, -2)) / math.sqrt(D), (j < P) | (j - P <= last))
        out[b] = (p @ vs).flatten(0, 1).transpose(0, 1)
        lse[b] = row_lse.flatten(0, 1).t()
    return out.to(DTYPES[case["dtype"]]), lse


# ------------------------------------------------------------------------------------------------ work
def _pairs(case):
    """Seen (query, key) pairs of one head."""
    if case["kind"] == "shared":
        n = case["n"]
        return sum(n * case["P"] + sum(max(0, m - n + i + 1) for i in range(n)) for m in _numbers(case["lens"]))
    total = 0
    for n, m in zip(*_lengths(case)):
        if not case["causal"]:
            total += n * m
        else:
            rows = min(n, m)      # the last `rows` queries see m - rows + 1 .. m keys
            total += rows * (m - rows) + rows * (rows + 1) // 2
    return total


def work(case):
    H, Hk, D = case["H"], case["Hk"], case["D"]
    pairs = _pairs(case) * H * D
    if case["kind"] == "shared":
        lens = _numbers(case["lens"])
        rows = len(lens) * case["n"] * H
        return {"bytes": rows * (4 * D + 4) + (case["P"] + sum(lens)) * Hk * D * 4, "flops": 4 * pairs}
    lq, lk = _lengths(case)
    rows, keys = sum(lq) * H, sum(lk) * Hk
    if case["train"]:       # q, dout, out, dq; k, v, dk, dv
        return {"bytes": rows * D * 8 + keys * D * 8, "flops": 14 * pairs}
    return {"bytes": rows * (D * 4 + 4) + keys * D * 4, "flops": 4 * pairs}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _attend64(q, k, v, mask, extra=None):
    """One head: softmax over the True columns of mask [n, m] of q k^T / sqrt(D) + extra, times v; (o, lse)."""
    s = q.mm(k.t()) * q.shape[1] ** -0.5
    if extra is not None:
        s = s + extra
    s = s.masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(s, 1)
    w = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[:, None])
    return w.mm(v), lse


def exact(case, seed):
    t = _inputs(case, seed)
    H, Hk = case["H"], case["Hk"]
    G = H // Hk
    if case["kind"] == "shared":
        n, P = case["n"], case["P"]
        out = torch.zeros(t["q"].shape, device="cuda", dtype=torch.float64)
        lse = torch.zeros(t["q"].shape[:3], device="cuda", dtype=torch.float64)
        for c in range(Hk):
            kp, vp = t["kp"][:, c].double(), t["vp"][:, c].double()
            for b, m in enumerate(_numbers(case["lens"])):
                keys = torch.cat([kp, t["k"][b, :m, c].double()])
                vals = torch.cat([vp, t["v"][b, :m, c].double()])
                mask = torch.ones(n, P + m, dtype=torch.bool, device="cuda").tril(P + m - n)
                mask[:, :P] = True
                rows = t["q"][b, :, c * G:(c + 1) * G].double().reshape(n * G, -1)       # (token, head in group)
                o, l = _attend64(rows, keys, vals, mask.repeat_interleave(G, 0))
                out[b, :, c * G:(c + 1) * G] = o.reshape(n, G, -1)
                lse[b, :, c * G:(c + 1) * G] = l.reshape(n, G)
        return out, lse
    lq, lk = _lengths(case)
    out = torch.zeros(t["q"].shape, device="cuda", dtype=torch.float64)
    lse = torch.full(t["q"].shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    names = [x for x in ("q", "k", "v", "bias") if x in t]
    grads = {x: torch.zeros(t[x].shape, device="cuda", dtype=torch.float64) for x in names} if case["train"] else {}
    at_q, at_k = _starts(lq), _starts(lk)
    for b, (n, m) in enumerate(zip(lq, lk)):
        if n == 0 or m == 0:
            continue
        rows, cols = slice(at_q[b], at_q[b + 1]), slice(at_k[b], at_k[b + 1])
        mask = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if case["causal"]:
            mask = mask.tril(m - n)
        if case["buckets"]:
            table = torch.tensor([_bucket(d, case["buckets"], not case["causal"]) for d in range(-m, n + m + 1)],
                                 device="cuda")
            offset = torch.arange(m, device="cuda")[None] - torch.arange(m - n, m, device="cuda")[:, None]
            place = table[offset + m]
        for h in range(H):
            x = [t["q"][rows, h], t["k"][cols, h // G], t["v"][cols, h // G]]
            x = [y.double().requires_grad_(case["train"]) for y in x]
            extra = None
            if case["buckets"]:
                w = t["bias"][:, h].double().requires_grad_(case["train"])
                extra = w[place]
            o, l = _attend64(*x, mask, extra)
            out[rows, h], lse[rows, h] = o.detach(), l.detach()
            if case["train"]:
                gr = torch.autograd.grad(o, x + ([w] if case["buckets"] else []), t["dout"][rows, h].double())
                grads["q"][rows, h] = gr[0]
                grads["k"][cols, h // G] += gr[1]
                grads["v"][cols, h // G] += gr[2]
                if case["buckets"]:
                    grads["bias"][:, h] += gr[3]
    return (out, *grads.values()) if case["train"] else (out, lse)
