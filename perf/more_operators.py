"""Norms and position rotation of queries and keys, a paged cache that they are appended to (16 or 4 bits), and attention over
it: cases, plain forms and 64-bit results.

Where `own` is false, `run` computes the operators in plain torch operations; where it is true it calls `norm_rotate`,
`append_paged`, `paged_rows` and `paged_attention` as a program does. Lengths are part of a case (comma-separated texts, one
number a sequence), so the work of a case follows from it alone; every input value comes from the seed.

A sequence's `keys` are all its tokens, `lens` how many of them are new: the last ones. Token i of n new ones among m stands at
position m - n + i, is held in row position % page of page pages[sequence, position // page], and sees the keys up to its own.

4 bits: 32 channels share a power of two s, the smallest with max |x| <= 7 s (bf16: 2^-120 .. 2^120, fp16: 2^-13 .. 2^13), held
as its exponent + 127 in a byte; a value is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times s, the nearest to x, ties to the
even code; channel 2 i is in the low half of byte i. x is the normed and rotated value rounded to float32, not to the token
type.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS, THETA = 1e-6, 10000.0


def listed():
    return [
        # queries and keys of four single tokens, a quarter of the channels' pairs rotated: launches and host work count
        dict(name="rotate_tokens", kind="rotate", lens="1,1,1,1", grid="", H=8, Hk=2, D=64, R=32, halves=True, norm=True,
             dtype="fp16", train=False),
        # a video's tokens, three axes of positions, many heads: bandwidth
        dict(name="rotate_clip", kind="rotate", lens="", grid="21,30,52", H=40, Hk=40, D=128, R=128, halves=False, norm=True,
             dtype="bf16", train=False),
        # a training step over packed sequences, three query heads to a key head
        dict(name="rotate_train", kind="rotate", lens="4096,1000,3,2049,6553,1", grid="", H=24, Hk=8, D=128, R=128,
             halves=True, norm=True, dtype="bf16", train=True),
        # one generated token for each of 48 requests goes into the cache
        dict(name="append_tokens", kind="append", lens=",".join(["1"] * 48),
             keys=",".join(str(1 + 331 * i % 4000) for i in range(48)), H=32, Hk=8, D=128, R=128, halves=True, norm=True,
             dtype="bf16", page=64, bits=16, pad=0),
        # whole prompts, small pages, rotation without a norm, some rows of padding behind them
        dict(name="append_prompts", kind="append", lens="4096,37,2011,1,777,6000", keys="4096,37,2011,1,777,6000", H=32, Hk=8,
             D=128, R=128, halves=False, norm=False, dtype="fp16", page=16, bits=16, pad=22),
        # pieces of prompts behind longer histories, held in 4 bits
        dict(name="append4_prompts", kind="append", lens="4096,1000,600", keys="32760,9000,600", H=40, Hk=8, D=128, R=128,
             halves=True, norm=True, dtype="bf16", page=64, bits=4, pad=0),
        # one token for four short requests: the smallest attention call
        dict(name="attend_small", kind="attend", lens="1,1,1,1", keys="129,1,77,300", H=8, Hk=2, D=64, dtype="bf16", page=16,
             bits=16, pad=0),
        # single tokens against long histories of very different lengths: bandwidth, one of them half of it
        dict(name="attend_long", kind="attend", lens="1,1,1,1,1,1,1,1", keys="32760,4097,75600,1209,16384,20011,513,9000",
             H=40, Hk=8, D=128, dtype="fp16", page=64, bits=16, pad=0),
        # pieces of prompts appended to what is there already, beside a single token
        dict(name="attend_chunks", kind="attend", lens="256,512,31,1", keys="9000,512,4111,2600", H=24, Hk=8, D=128,
             dtype="bf16", page=32, bits=16, pad=3),
        # a token for each of 48 requests, cache of 4 bits
        dict(name="attend4_tokens", kind="attend", lens=",".join(["1"] * 48),
             keys=",".join(str(1 + 1331 * i % 16000) for i in range(48)), H=32, Hk=8, D=128, dtype="bf16", page=64, bits=4,
             pad=0),
        # the long histories in 4 bits
        dict(name="attend4_long", kind="attend", lens="1,1,1,1,1,1,1,1", keys="32760,4097,75600,1209,16384,20011,513,9000",
             H=40, Hk=8, D=128, dtype="fp16", page=16, bits=4, pad=0),
        # pieces of prompts and single tokens over 4 bits
        dict(name="attend4_chunks", kind="attend", lens="700,64,1,1,2048", keys="16384,5000,8000,75600,2048", H=32, Hk=8,
             D=128, dtype="bf16", page=128, bits=4, pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= 2.3e11 and w["bytes"] <= 1.4e9:
            return case


def _draw(rng):
    kind = rng.choice(["rotate", "rotate", "append", "append", "tokens", "tokens", "chunks"])
    D = rng.choice([64, 128, 128])
    Hk = rng.choice([1, 2, 3, 5, 8])
    case = dict(H=Hk * rng.choice([1, 1, 2, 3, 4, 5, 8]), Hk=Hk, D=D, dtype=rng.choice(["bf16", "fp16"]))
    turn = dict(R=rng.choice([D, D, D // 2, 16, 48]), halves=rng.random() < 0.5, norm=rng.random() < 0.7)
    if kind == "rotate":
        case.update(turn, kind=kind, lens="", grid="", train=rng.random() < 0.6)
        if rng.random() < 0.4:
            case.update(R=D, grid=",".join(str(_log(rng, 1, top)) for top in (21, 45, 80)))
        else:
            case["lens"] = ",".join(str(_log(rng, 1, 9000)) for _ in range(_log(rng, 1, 10)))
        return case
    case.update(page=rng.choice([16, 32, 64, 64, 128, 256]), bits=rng.choice([16, 4]), pad=rng.choice([0, 0, 1, 50]))
    if kind == "tokens":
        B = _log(rng, 1, 200)
        return dict(case, kind="attend", lens=",".join(["1"] * B), keys=",".join(str(_log(rng, 1, 40000)) for _ in range(B)))
    lens = [_log(rng, 1, 5000) for _ in range(_log(rng, 1, 10))]
    if rng.random() < 0.3:
        lens = [rng.choice([1, 2, 5, 16])] * _log(rng, 1, 64)
    keys = [n + (rng.random() < 0.7) * _log(rng, 1, 20000) for n in lens]
    case.update(lens=",".join(map(str, lens)), keys=",".join(map(str, keys)))
    return dict(case, **turn, kind="append") if kind == "append" else dict(case, kind="attend")


# ------------------------------------------------------------------------------------------------ inputs
def _numbers(text):
    return [int(x) for x in text.split(",")]


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _tokens(case):
    if case["kind"] == "rotate" and case["grid"]:
        return math.prod(_numbers(case["grid"]))
    return sum(_numbers(case["lens"])) + case.get("pad", 0)


def _turns(positions, dim):
    """(cos, sin) of positions times the dim / 2 frequencies, float32 [P, dim / 2, 2] from angles in 64 bits."""
    freq = THETA ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    angle = positions.double()[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _grid_turns(grid, dim):
    """A row each for the points of a grid in order; the channels are shared out among its axes, the first one the most."""
    rest = dim // 6 * 2
    at = torch.cartesian_prod(*(torch.arange(n, device="cuda") for n in grid)).reshape(-1, 3)
    return torch.cat([_turns(at[:, i], d) for i, d in enumerate((dim - 2 * rest, rest, rest))], 1)


SMALLEST, LARGEST = {"bf16": -120, "fp16": -13}, {"bf16": 120, "fp16": 13}


def _power(e):
    """2^e in float64, from the exponent's bits: exact, which powers by a function need not be."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _quantise(x, dtype):
    """(codes uint8 [..., D / 2], exponents + 127 uint8 [..., D / 32]) of float32 x [..., D]."""
    x = x.unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    frac, e = torch.frexp(top)                        # top = frac 2^e, 0.5 <= frac < 1
    e = torch.where(frac > 0.875, e - 2, e - 3)       # 7 s >= top: s = 2^(e - 3) holds up to 0.875 2^e
    e = torch.where(top == 0, SMALLEST[dtype], e).clamp(SMALLEST[dtype], LARGEST[dtype])
    y = x.double() * _power(-e)[..., None]            # exact
    a = y.abs()
    borders = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))
    code = torch.zeros_like(a, dtype=torch.uint8)
    for border, up in borders:                        # between an even and an odd code the even one takes the border
        code += (a >= border if up else a > border).to(torch.uint8)
    code |= (torch.signbit(y) & (code > 0)).to(torch.uint8) << 3
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] | code[..., 1] << 4, (e + 127).to(torch.uint8)


def _inputs(case, seed):
    """The tensors of a case by name."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, H, Hk, D, T = DTYPES[case["dtype"]], case["H"], case["Hk"], case["D"], _tokens(case)
    rnd = lambda *shape, std=1.0: std * torch.randn(*shape, device="cuda", generator=g)
    t = {}
    if case["kind"] != "attend":
        # queries, keys and values are column ranges of one projection's rows; the channels differ in size
        rows = rnd(T, H + 2 * Hk, D, std=1.5).mul_(torch.exp(rnd(D, std=0.3))).to(dt)
        t.update(q=rows[:, :H], k=rows[:, H:H + Hk], v=rows[:, H + Hk:])
        if case["norm"]:
            t.update(qw=(1 + rnd(D, std=0.2)).to(dt), kw=(1 + rnd(D, std=0.2)).to(dt))
        if case.get("train"):
            t.update(dq=rnd(T, H, D).to(dt), dk=rnd(T, Hk, D).to(dt))
    else:
        t["q"] = rnd(T, H, D, std=1.5).to(dt)
    if case["kind"] == "rotate":
        lens = [] if case["grid"] else _numbers(case["lens"])
        if case["grid"]:
            t["table"] = _grid_turns(_numbers(case["grid"]), case["R"])
        else:
            t["table"] = _turns(torch.arange(max(lens), device="cuda"), case["R"])
            t["positions"] = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in lens])
        return t
    lens, keys, page = _numbers(case["lens"]), _numbers(case["keys"]), case["page"]
    if case["kind"] == "append":
        t["table"] = _turns(torch.arange(max(keys), device="cuda"), case["R"])
    # the pages of all sequences are spread over the cache in any order; entries that no key needs hold -1
    need = [-(-m // page) for m in keys]
    order = torch.randperm(sum(need) + 3, device="cuda", generator=g).to(torch.int32)
    t["pages"] = torch.full((len(keys), max(need)), -1, device="cuda", dtype=torch.int32)
    for b, (at, n) in enumerate(zip(_starts(need), need)):
        t["pages"][b, :n] = order[at:at + n]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    t.update(lens=ints(keys), cu=ints(_starts(lens)))
    for name in "kv":
        x = rnd(len(order), Hk, page, D)
        if case["bits"] == 4:
            t[name + "c"], t[name + "s"] = _quantise(x, case["dtype"])
        else:
            t[name + "c"] = x.to(dt)
    return t


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if case.get("train"):
        for name in ("q", "k", "qw", "kw"):
            if name in state:
                state[name] = state[name].detach().requires_grad_()
    return state


# ------------------------------------------------------------------------------------------------ passes
def run(state):
    case = state["case"]
    if not own:
        return {"rotate": _plain_rotate, "append": _plain_append, "attend": _plain_attend}[case["kind"]](state)
    from self_trainable_or_free_attn_amd import PagedCache, append_paged, norm_rotate, paged_attention, paged_rows
    if case["kind"] == "rotate":
        out = norm_rotate(state["q"], state["k"], state.get("qw"), state.get("kw"), state["table"], state.get("positions"),
                          eps=EPS, halves=case["halves"])
        if not case["train"]:
            return out
        leaves = [state[n] for n in ("q", "k", "qw", "kw") if n in state]
        return (*out, *torch.autograd.grad(out, leaves, (state["dq"], state["dk"])))
    cache = PagedCache(state["kc"], state["vc"], state.get("ks"), state.get("vs"))
    if case["kind"] == "attend":
        return paged_attention(state["q"], cache, state["pages"], state["lens"], state["cu"], return_lse=True)
    q = append_paged(cache, state["k"], state["v"], state["pages"], state["lens"], state["cu"], q=state["q"],
                     q_weight=state.get("qw"), k_weight=state.get("kw"), table=state["table"], eps=EPS,
                     halves=case["halves"])
    if case["bits"] == 16:
        return q, cache.k, cache.v
    return q, *paged_rows(cache, state["pages"], state["lens"], state["cu"], rows=_tokens(case), dtype=q.dtype)


def _apart(x, R, halves):
    """The first and the second channel of each rotated pair."""
    return (x[..., :R // 2], x[..., R // 2:R]) if halves else (x[..., 0:R:2], x[..., 1:R:2])


def _turn(x, cs, halves, back=False):
    """x [T, H, D] rotated by the angles cs [T, R / 2, 2] (back: by their negatives)."""
    R = 2 * cs.shape[1]
    c, s = cs[:, None, :, 0], -cs[:, None, :, 1] if back else cs[:, None, :, 1]
    a, b = _apart(x, R, halves)
    first, second = a * c - b * s, a * s + b * c
    pair = torch.cat([first, second], -1) if halves else torch.stack([first, second], -1).flatten(-2)
    return torch.cat([pair, x[..., R:]], -1)


def _unit(x):
    """x over its root mean square, and the reciprocal of that."""
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x * r, r


def _plain_rotate(state):
    case, halves, train = state["case"], state["case"]["halves"], state["case"]["train"]
    cs = state["table"]
    if "positions" in state:
        cs = cs[state["positions"].long()]
    out, grads, weights = [], [], []
    for name in "qk":
        x = state[name].detach().float()
        w = state[name + "w"].detach().float() if case["norm"] else None
        if case["norm"]:
            x, r = _unit(x)
        out.append(_turn(x * w if case["norm"] else x, cs, halves).to(state[name].dtype))
        if not train:
            continue
        g = _turn(state["d" + name].float(), cs, halves, back=True)
        if case["norm"]:
            weights.append((g * x).sum((0, 1), dtype=torch.float64).to(state[name].dtype))
            g = g * w
            g = r * (g - x * (g * x).mean(-1, keepdim=True))
        grads.append(g.to(state[name].dtype))
    return (*out, *grads, *weights)


VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _values(codes, scales):
    """The float32 values of 4-bit rows."""
    table = torch.tensor(VALUES + tuple(-x for x in VALUES), device="cuda")
    x = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()]
    return (x.unflatten(-1, (-1, 32)) * _power(scales.int() - 127).float()[..., None]).flatten(-2)


def _places(state):
    """Of every token of the sequences: its position, and the page and row that hold it."""
    case, cu = state["case"], state["cu"].long()
    at = torch.arange(_tokens(case) - case["pad"], device="cuda")
    b = torch.searchsorted(cu[1:], at, right=True)
    position = state["lens"].long()[b] + at - cu[b + 1]
    return position, state["pages"].long()[b, position // case["page"]], position % case["page"]


def _plain_append(state):
    case, dt = state["case"], state["q"].dtype
    position, page, row = _places(state)
    n = len(position)
    cs = state["table"][position].double()
    turned = []
    for name in "qk":       # (in 64 bits: a key's 4-bit code may stand next to a border)
        x = state[name][:n].double()
        if case["norm"]:
            x = _unit(x)[0] * state[name + "w"].double()
        turned.append(_turn(x, cs, case["halves"]).float())
    q = torch.zeros_like(state["q"], memory_format=torch.contiguous_format)
    q[:n] = turned[0].to(dt)
    if case["bits"] == 16:
        state["kc"][page, :, row] = turned[1].to(dt)
        state["vc"][page, :, row] = state["v"][:n]
        return q, state["kc"], state["vc"]
    out = []
    for name, x in (("k", turned[1]), ("v", state["v"][:n].float())):
        codes, scales = state[name + "c"], state[name + "s"]
        codes[page, :, row], scales[page, :, row] = _quantise(x, case["dtype"])
        rows = torch.zeros(_tokens(case), case["Hk"], case["D"], device="cuda", dtype=dt)
        rows[:n] = _values(codes[page, :, row], scales[page, :, row]).to(dt)
        out.append(rows)
    return q, *out


MOST_SCORES = 1 << 29


def _plain_attend(state):
    case, page = state["case"], state["case"]["page"]
    H, Hk, D = case["H"], case["Hk"], case["D"]
    q = state["q"].float()
    out = torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, device="cuda")
    lens, keys = _numbers(case["lens"]), _numbers(case["keys"])
    for b, (at, n, m) in enumerate(zip(_starts(lens), lens, keys)):
        held = state["pages"][b, :-(-m // page)].long()
        kv = []
        for name in "kv":
            x = state[name + "c"][held]
            x = _values(x, state[name + "s"][held]) if case["bits"] == 4 else x.float()
            kv.append(x.transpose(0, 1).flatten(1, 2)[:, None, :m])                   # [Hk, 1, m, D]
        j = torch.arange(m, device="cuda")
        step = max(1, MOST_SCORES // (H * m))
        for r in range(0, n, step):
            rows = q[at + r:at + min(n, r + step)]
            x = rows.unflatten(1, (Hk, H // Hk)).permute(1, 2, 0, 3)                  # [Hk, G, rows, D]
            s = (x @ kv[0].transpose(-1, -2)) / math.sqrt(D)
            last = m - n + r + torch.arange(len(rows), device="cuda")
            s = torch.where(j <= last[:, None], s, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True)
            to = slice(at + r, at + r + len(rows))
            out[to] = (p @ kv[1] / total).flatten(0, 1).transpose(0, 1)
            lse[to] = (top + torch.log(total))[..., 0].flatten(0, 1).t()
    return out.to(state["q"].dtype), lse


# ------------------------------------------------------------------------------------------------ work
def work(case):
    H, Hk, D, T = case["H"], case["Hk"], case["D"], _tokens(case)
    if case["kind"] == "rotate":
        # every row read and written, training: the incoming gradient read and the outgoing one written as well; the angles
        points = T if case["grid"] else max(_numbers(case["lens"]))
        rows = T * (H + Hk) * D
        return {"bytes": rows * (8 if case["train"] else 4) + points * case["R"] * 4, "flops": rows * (20 if case["train"] else 7)}
    held = D * 2 if case["bits"] == 16 else D // 2 + D // 32
    lens, keys = _numbers(case["lens"]), _numbers(case["keys"])
    if case["kind"] == "append":
        n = sum(lens)
        angles = sum(lens) * case["R"] * 4
        moved = T * H * D * 2 + n * (H + 2 * Hk) * D * 2 + n * 2 * Hk * held
        if case["bits"] == 4:      # the new rows as they are held, read back
            moved += n * 2 * Hk * held + T * 2 * Hk * D * 2
        return {"bytes": moved + angles, "flops": n * (H + 2 * Hk) * D * 7}
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(lens, keys))
    return {"bytes": T * H * (4 * D + 4) + sum(keys) * Hk * 2 * held, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _rotated64(x, w, cs, halves):
    """The operator in complex numbers: a pair is a number, its angle a factor of modulus 1."""
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
    R = 2 * cs.shape[1]
    turn = torch.view_as_complex(cs.double().contiguous())[:, None]
    if halves:
        z = torch.complex(x[..., :R // 2], x[..., R // 2:R]) * turn
        return torch.cat([z.real, z.imag, x[..., R:]], -1)
    z = torch.view_as_complex(x[..., :R].unflatten(-1, (-1, 2)).contiguous()) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), x[..., R:]], -1)


def _powers64(e):
    """2^e for whole e from -127 to 128."""
    return torch.tensor([2.0 ** i for i in range(-127, 129)], dtype=torch.float64, device="cuda")[e.long() + 127]


def _held64(x, dtype):
    """The 4-bit values nearest to x, by steps of a power of two: 0.5 s below 2 s, s from there to 4 s, 2 s above."""
    g = x.unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    s = _powers64(torch.log2(top / 7).ceil().clamp(SMALLEST[dtype], LARGEST[dtype]))
    s = torch.where(top > 7 * s, 2 * s, torch.where(top <= 3.5 * s, s / 2, s))      # (a logarithm that is a last bit off)
    s = s.clamp(2.0 ** SMALLEST[dtype], 2.0 ** LARGEST[dtype])
    a = g.abs() / s
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.sign(g) * (torch.round(a / step) * step).clamp(max=6) * s).flatten(-2)


def _decoded64(codes, scales):
    """Sign, two bits of exponent, one of mantissa."""
    n = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    e, m = n // 2 % 4, (n % 2).double()
    a = torch.where(e == 0, m / 2, (1 + m / 2) * _powers64(e - 1)) * (1 - 2 * (n // 8)).double()
    return a * _powers64(scales.long() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "rotate":
        cs = t["table"] if case["grid"] else t["table"].index_select(0, t["positions"].long())
        out, grads, weights = [], [], []
        for name in "qk":
            x = t[name].double()
            w = t[name + "w"].double() if case["norm"] else None
            leaves = [y.requires_grad_(case["train"]) for y in (x, w) if y is not None]
            y = _rotated64(*leaves, *([] if case["norm"] else [None]), cs, case["halves"])
            out.append(y.detach())
            if case["train"]:
                g = torch.autograd.grad(y, leaves, t["d" + name].double())
                grads.append(g[0])
                weights += g[1:]
            del x, y
        return (*out, *grads, *weights)
    lens, keys, page, Hk = _numbers(case["lens"]), _numbers(case["keys"]), case["page"], case["Hk"]
    if case["kind"] == "append":
        n = sum(lens)
        position = torch.cat([torch.arange(m - i, m, device="cuda") for i, m in zip(lens, keys)])
        cs = t["table"][position]
        q, k = (_rotated64(t[x][:n], t.get(x + "w"), cs, case["halves"]) for x in "qk")
        padded = lambda x: torch.cat([x, x.new_zeros(case["pad"], *x.shape[1:])])
        if case["bits"] == 4:
            return padded(q), padded(_held64(k, case["dtype"])), padded(_held64(t["v"][:n].double(), case["dtype"]))
        kc, vc, v = t["kc"].double(), t["vc"].double(), t["v"].double()
        for b, (at, i, m) in enumerate(zip(_starts(lens), lens, keys)):
            p = torch.arange(m - i, m, device="cuda")
            held = t["pages"][b].long()[torch.div(p, page, rounding_mode="floor")]
            kc[held, :, p % page], vc[held, :, p % page] = k[at:at + i], v[at:at + i]
        return padded(q), kc, vc
    out = torch.zeros(t["q"].shape, device="cuda", dtype=torch.float64)
    lse = torch.full(t["q"].shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    G = case["H"] // Hk
    for b, (at, n, m) in enumerate(zip(_starts(lens), lens, keys)):
        held = t["pages"][b, :(m + page - 1) // page].long()
        mask = torch.ones(n, m, dtype=torch.bool, device="cuda").tril(m - n)
        for h in range(Hk):
            k, v = (_decoded64(t[x + "c"][held, h], t[x + "s"][held, h]) if case["bits"] == 4 else t[x + "c"][held, h].double()
                    for x in "kv")
            k, v = k.flatten(0, 1)[:m], v.flatten(0, 1)[:m]
            for i in range(h * G, h * G + G):
                s = (t["q"][at:at + n, i].double().mm(k.t()) * case["D"] ** -0.5).masked_fill(~mask, -math.inf)
                lse[at:at + n, i] = torch.logsumexp(s, 1)
                out[at:at + n, i] = torch.softmax(s, 1).mm(v)
    return out, lse
