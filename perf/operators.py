"""What the cache operators over 4-bit pages and the windowed attention with sinks compute, and real
calls of them to measure.

Three operators, each over rows of keys and values [rows][kv_heads][head_dim] (f32 in, f32 out):

* write: rows are quantised to 4-bit codes as they go into the cache, and read back as f32;
* attend: decode attention, one query token per sequence, over a cache held in 4 bits; with `append`
  the token's own row is quantised into the cache by the same call;
* sinks: decode attention that sees the last `window` rows and the first `sinks` rows, over pages
  held in 4 bits, bf16 or f32.

The 4-bit format. A head row is cut into groups of 32 values x. Rows at even positions count up from
the group's minimum, rows at odd positions down from its maximum: with y = x on even rows, y = -x on odd
ones,
    bias  = bf16(min y)
    step  = bf16(max((max y - bias) / 15, 2^-40, 2^(e-16))),  2^e the power of two at or below the
            largest (max y - bias) / 15 of the head row
    code  = nearest((y - bias) / step), ties to even, kept within 0..15
and the row reads back as (code * step + bias), negated on odd rows. Every rounding is of the exact value.

`own` chooses between the plain form (torch operations) and the calls of this package.
"""
import math

import torch

own = False

GROUP = 32
PAGES = {"f32": 0, "bf16": 1, "u4": 3}


# ---- cases ----------------------------------------------------------------------------------------
def listed():
    return [
        # one token's row of one layer: latency only
        dict(name="write_token", op="write", rows=1, offset=1000, kv_heads=8, hd=128),
        # a chunk of a prompt that starts and ends inside a page, large heads
        dict(name="write_chunk_odd", op="write", rows=333, offset=7, kv_heads=2, hd=256),
        # one layer of a prompt
        dict(name="write_prompt", op="write", rows=4096, offset=0, kv_heads=8, hd=128),
        # a long prompt on a head-sharded device
        dict(name="write_prompt_long", op="write", rows=32768, offset=0, kv_heads=4, hd=128),
        # the first tokens of an answer
        dict(name="attend_short", op="attend", seqs=1, rows=77, spread=1.0, q_heads=32, kv_heads=8, hd=128, append=False),
        # one long conversation
        dict(name="attend_long", op="attend", seqs=1, rows=32768, spread=1.0, q_heads=32, kv_heads=4, hd=128, append=False),
        # a decode step of two sequences, the new rows written by the same call
        dict(name="attend_step_hd256", op="attend", seqs=2, rows=16001, spread=1.0, q_heads=16, kv_heads=2, hd=256, append=True),
        # many conversations of very different lengths
        dict(name="attend_uneven", op="attend", seqs=24, rows=20000, spread=0.01, q_heads=32, kv_heads=8, hd=128, append=False),
        # a full batch of long contexts: the largest
        dict(name="attend_batch", op="attend", seqs=8, rows=32768, spread=1.0, q_heads=32, kv_heads=4, hd=128, append=False),
        # a local layer of a small request, f32 pages
        dict(name="sinks_f32_small", op="sinks", pages="f32", seqs=1, rows=500, spread=1.0, q_heads=8, kv_heads=2, hd=128,
             window=100, sinks=5),
        # local layers of a batch with bf16 pages
        dict(name="sinks_bf16", op="sinks", pages="bf16", seqs=16, rows=30000, spread=0.3, q_heads=32, kv_heads=4, hd=128,
             window=4096, sinks=4),
        # endless streams over a small cache
        dict(name="sinks_u4_streams", op="sinks", pages="u4", seqs=64, rows=9000, spread=0.5, q_heads=16, kv_heads=2, hd=256,
             window=2000, sinks=20),
    ]


LARGEST = 8 * 32768 * 4 * 128     # cached values of the largest listed case, K


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write", "attend", "sinks"))
    hd = rng.choice((64, 96, 128, 128, 128, 256, 256))
    kv_heads = rng.choice((1, 2, 4, 8))
    if op == "write":
        rows = _log_int(rng, 1, min(32768, LARGEST // (8 * kv_heads * hd)))
        return dict(op=op, rows=rows, offset=rng.randrange(0, 200), kv_heads=kv_heads, hd=hd)
    gqa = rng.choice((1, 2, 4, 5, 8, 8))
    seqs = _log_int(rng, 1, 64)
    # the CUDA-core kernel of the other head sizes re-reads a page per query head: such shapes are small models
    most = LARGEST if hd in (128, 256) else LARGEST // 16
    rows = _log_int(rng, 1, max(2, min(40000, most // (seqs * kv_heads * hd))))
    case = dict(op=op, seqs=seqs, rows=rows, spread=rng.choice((1.0, 1.0, 0.5, 0.05)), q_heads=gqa * kv_heads, kv_heads=kv_heads,
                hd=hd)
    if op == "attend":
        return dict(case, append=rng.random() < 0.3)
    pages = rng.choice(("u4", "u4", "bf16", "f32"))
    if pages == "f32":
        case["rows"] = max(1, rows // 4)
    return dict(case, pages=pages, window=_log_int(rng, 1, 8192), sinks=rng.choice((0, 1, 4, 4, 16, 37, 128)))


def _lens(case):
    """Rows of every sequence: the longest first, the others down to `spread` of it, spaced evenly in the logarithm."""
    n, rows = case["seqs"], case["rows"]
    low = max(1.0, rows * case["spread"])
    return [max(1, int(round(rows * (low / rows) ** (i / (n - 1))))) for i in range(n)] if n > 1 else [rows]


def _visible(case, length):
    """(rows at the head, first row of the tail) that the attention sees."""
    start = max(0, length - case["window"]) if case["op"] == "sinks" else 0
    return min(case.get("sinks", 0), start), start


# ---- inputs ---------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)


def _rows(case, seed):
    """K and V rows: keys with channels of their own mean and spread (as after a norm and a rotation), values without."""
    g = _generator(seed)
    shape = (case["rows"], case["kv_heads"], case["hd"])
    mean = 0.8 * torch.randn(shape[1:], device="cuda", generator=g)
    spread = 0.4 + torch.rand(shape[1:], device="cuda", generator=g)
    return mean + spread * torch.randn(shape, device="cuda", generator=g), torch.randn(shape, device="cuda", generator=g)


def _sequences(case, seed):
    """Queries [seqs][q_heads][hd], and a function that makes K and V rows [rows of i][kv_heads][hd] of sequence i. The
    first four keys draw attention, as the first tokens of a text do."""
    g = _generator(seed)
    heads, hd = case["kv_heads"], case["hd"]
    toward = 0.35 * torch.randn((heads, hd), device="cuda", generator=g)
    mean = 0.5 * torch.randn((heads, hd), device="cuda", generator=g)
    spread = 0.4 + torch.rand((heads, hd), device="cuda", generator=g)
    q = torch.randn((case["seqs"], heads, case["q_heads"] // heads, hd), device="cuda", generator=g) + toward[:, None, :]
    lens = _lens(case)

    def rows_of(i):
        gi = _generator(int(seed) * 1009 + 17 * i + 3)
        k = mean + spread * torch.randn((lens[i], heads, hd), device="cuda", generator=gi)
        v = torch.randn((lens[i], heads, hd), device="cuda", generator=gi)
        k[:4] += 3.0 * toward
        return k, v

    return q.reshape(case["seqs"], case["q_heads"], hd).contiguous(), rows_of, lens


# ---- the plain form ---------------------------------------------------------------------------------
def _bf16_of(x):
    """Nearest bf16 value (ties to even) of f64 values, rounded once."""
    bits = x.view(torch.int64)
    bits = bits + (1 << 44) - 1 + ((bits >> 45) & 1)
    return (bits >> 45 << 45).view(torch.float64)


def _quantise(x, row0):
    """Codes (u8), signed step and signed bias (f32) of rows x [rows][heads][hd] that start at position row0."""
    rows, heads, hd = x.shape
    odd = ((torch.arange(rows, device=x.device) + row0) % 2).view(rows, 1, 1, 1)
    sign = (1 - 2 * odd).double()
    y = x.view(rows, heads, hd // GROUP, GROUP).double() * sign
    bias = _bf16_of(y.amin(-1, keepdim=True))
    raw = (y.amax(-1, keepdim=True) - bias) / 15
    widest = raw.amax(2, keepdim=True).clamp_min(2.0 ** -40)
    floor = torch.ldexp(torch.ones_like(widest), torch.frexp(widest)[1] - 17)
    step = _bf16_of(torch.maximum(raw, floor).clamp_min(2.0 ** -40))
    code = torch.round((y - bias) / step).clamp(0, 15).to(torch.uint8)
    return code, (step * sign).float(), (bias * sign).float()


def _read(code, step, bias):
    """The f32 values that codes stand for; code * step has at most 12 bits, so only the sum rounds."""
    return (code.float() * step + bias).flatten(-2)


def _pad(parts, most):
    return torch.stack([torch.nn.functional.pad(p, (0, 0) * (p.dim() - 1) + (0, most - p.shape[0])) for p in parts])


def _plain_pages(case, rows_of, lens):
    """The cache of the plain form: {"k": [...], "v": [...]}, every array [seqs][longest][kv_heads]..."""
    pages, most = case.get("pages", "u4"), max(lens)
    kept = {"k": [], "v": []}
    for i in range(case["seqs"]):
        for name, x in zip("kv", rows_of(i)):
            kept[name].append(_quantise(x, 0) if pages == "u4" else (x.to(torch.bfloat16) if pages == "bf16" else x,))
    return {name: [_pad(list(p), most) for p in zip(*kept[name])] for name in "kv"}


def _plain_attention(q, k, v, lens, heads, sinks, starts):
    """softmax(q . k / sqrt(hd)) . v over the visible rows; k, v [seqs][rows][heads][hd], f32."""
    n, rows, _, hd = k.shape
    at = torch.arange(rows, device=q.device)
    seen = (at < lens[:, None]) & ((at < sinks[:, None]) | (at >= starts[:, None]))
    scores = (q.view(n, heads, -1, hd) * hd ** -0.5) @ k.permute(0, 2, 3, 1)
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = weights @ v.transpose(1, 2)
    return (out / weights.sum(-1, keepdim=True)).reshape(n, -1, hd)


def _plain_run(state):
    case = state["case"]
    if case["op"] == "write":
        return {"k": _read(*_quantise(state["k"], case["offset"])), "v": _read(*_quantise(state["v"], case["offset"]))}
    out = {}
    if case.get("append"):
        # the token's rows go into the cache (their position is odd or even by sequence, lengths differ)
        last = state["lens"] - 1
        for name in "kv":
            new = state["new_" + name]
            both = [_quantise(new, parity) for parity in (0, 1)]
            # row i of `new` was taken at position i + parity: choose the one whose parity is the true one
            pick = ((torch.arange(len(new), device=new.device) + last) % 2 == 0)
            for kept, even, odd in zip(state[name], *both):
                kept[state["seq"], last] = torch.where(pick.view(-1, *[1] * (even.dim() - 1)), even, odd)
            out["new_" + name] = _read(*(kept[state["seq"], last] for kept in state[name]))
    k, v = ((_read(*state[name]) if len(state[name]) > 1 else state[name][0].float()) for name in "kv")
    return dict(out, out=_plain_attention(state["q"], k, v, state["lens"], case["kv_heads"], state["sinks"], state["starts"]))


# ---- the package's calls ------------------------------------------------------------------------------
class _Device:
    """A tensor where the package expects a device buffer."""

    def __init__(self, tensor):
        self.tensor, self.ptr = tensor, tensor.data_ptr()


class _Cache:
    """The sequences of a case in the package's pages, closed with this object."""

    def __init__(self, case, lens, capacity):
        import saragossa_b200 as sg
        self.state = sg.DecodeResidentState(torch.cuda.current_device())
        pages = sum((n + 15) // 16 for n in capacity)
        self.pool = self.state.pool(1, case["kv_heads"], case["hd"], PAGES[case.get("pages", "u4")], pages, len(capacity),
                                    max(capacity))
        self.pool.shuffle_free_list(5)
        self.seqs = [self.pool.sequence(n) for n in capacity]
        self.kvs = [s.layer(0, case.get("q_heads", case["kv_heads"])) for s in self.seqs]
        for kv in self.kvs:
            kv.set_attention_sinks(case.get("sinks", 0))
        self.batch = sg.Batch(self.state, self.kvs)
        self.lens = lens

    def fill(self, i, k, v):
        torch.cuda.synchronize()
        self.kvs[i].encode_append_rows(_Device(k), _Device(v), len(k))
        self.state.sync()

    def __del__(self):
        for x in (getattr(self, "batch", None), *getattr(self, "seqs", ()), getattr(self, "pool", None), getattr(self, "state", None)):
            if x is not None:
                x.close()


def _own_run(state):
    case, cache = state["case"], state["cache"]
    # the stream that torch works on, where the results are read; its default stream has the handle 0, which the package
    # takes for its own stream, so that one goes by its other name (cudaStreamLegacy)
    stream = torch.cuda.current_stream().cuda_stream or 1
    if case["op"] == "write":
        kv = cache.kvs[0]
        kv.encode_truncate(case["offset"], stream=stream)
        kv.encode_append_rows(state["k"], state["v"], case["rows"], stream=stream)
        kv.encode_gather_rows_f32(state["k_out"], state["v_out"], case["offset"], case["rows"], stream=stream)
        return {"k": state["k_out"].tensor, "v": state["v_out"].tensor}
    if not case.get("append"):
        cache.batch.enqueue_attention(state["q"], state["out"], case.get("window", 0), stream=stream)
        return {"out": state["out"].tensor}
    cache.batch.enqueue_truncate([n - 1 for n in cache.lens], stream=stream)
    cache.batch.enqueue_step(state["new_k"], state["new_v"], state["q"], state["out"], stream=stream)
    for kv, n, (k, v) in zip(cache.kvs, cache.lens, state["rows_out"]):
        kv.encode_gather_rows_f32(k, v, n - 1, 1, stream=stream)
    return {"out": state["out"].tensor, "new_k": state["k_out"], "new_v": state["v_out"]}


# ---- what is measured ---------------------------------------------------------------------------------
def prepare(case, seed):
    if case["op"] == "write":
        k, v = _rows(case, seed)
        if not own:
            return {"case": case, "k": k, "v": v}
        total = case["offset"] + case["rows"]
        cache = _Cache(case, [total], [total])
        if case["offset"]:
            old = torch.zeros((case["offset"], case["kv_heads"], case["hd"]), device="cuda")
            cache.fill(0, old, old)
        return {"case": case, "cache": cache, "k": _Device(k), "v": _Device(v), "k_out": _Device(torch.empty_like(k)),
                "v_out": _Device(torch.empty_like(v))}
    q, rows_of, lens = _sequences(case, seed)
    append = case.get("append", False)
    if not own:
        at = [_visible(case, n) for n in lens]
        state = {"case": case, "q": q, **_plain_pages(case, rows_of, lens),
                 "lens": torch.tensor(lens, device="cuda"), "sinks": torch.tensor([a for a, _ in at], device="cuda"),
                 "starts": torch.tensor([b for _, b in at], device="cuda"), "seq": torch.arange(case["seqs"], device="cuda")}
        if append:
            state["new_k"], state["new_v"] = (torch.stack(x) for x in zip(*((k[-1], v[-1]) for k, v in map(rows_of, range(case["seqs"])))))
        return state
    cache = _Cache(case, lens, lens)
    new = []
    for i in range(case["seqs"]):
        k, v = rows_of(i)
        new.append((k[-1].clone(), v[-1].clone()))
        cache.fill(i, k, v)
    state = {"case": case, "cache": cache, "q": _Device(q), "out": _Device(torch.empty_like(q))}
    if append:
        state["new_k"], state["new_v"] = (_Device(torch.stack(x)) for x in zip(*new))
        state["k_out"], state["v_out"] = torch.empty_like(state["new_k"].tensor).flatten(1), torch.empty_like(state["new_v"].tensor).flatten(1)
        state["k_out"], state["v_out"] = (x.view(case["seqs"], case["kv_heads"], case["hd"]) for x in (state["k_out"], state["v_out"]))
        state["rows_out"] = [(_Device(state["k_out"][i]), _Device(state["v_out"][i])) for i in range(case["seqs"])]
    return state


def run(state):
    return _own_run(state) if own else _plain_run(state)


def work(case):
    hd, heads = case["hd"], case["kv_heads"]
    row = {"u4": hd // 2 + hd // GROUP * 4, "bf16": 2 * hd, "f32": 4 * hd}[case.get("pages", "u4")] * 2 * heads
    if case["op"] == "write":
        # the f32 rows in, the codes out; the codes in, the f32 values out
        return {"bytes": case["rows"] * (2 * row + 2 * 2 * 4 * hd * heads), "flops": 0}
    total = 0
    for n in _lens(case):
        sinks, start = _visible(case, n)
        total += sinks + n - start
    io = 2 * 4 * case["seqs"] * case["q_heads"] * hd
    if case.get("append"):
        io += case["seqs"] * (2 * row + 2 * 2 * 4 * hd * heads)
    return {"bytes": total * row + io, "flops": 4 * total * case["q_heads"] * hd}


# ---- the definition in 64 bits ------------------------------------------------------------------------
def _nearest(t):
    """Nearest whole number, ties to even, from floor alone."""
    low = torch.floor(t)
    rest = t - low
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2) == 1))
    return low + up


def _exact_bf16(x):
    mantissa, exponent = torch.frexp(x)
    return torch.ldexp(_nearest(mantissa * 256), exponent - 8)


def _exact_values(x, first):
    """What rows x [rows][heads][hd], written from position `first` on, read back as."""
    y = x.double().unflatten(-1, (-1, GROUP)).clone()
    flip = slice((first + 1) % 2, None, 2)     # the rows at odd positions
    y[flip] = -y[flip]
    bias = _exact_bf16(y.min(-1, keepdim=True).values)
    range15 = y.max(-1, keepdim=True).values - bias
    top = range15.max(2, keepdim=True).values / 15
    below = torch.exp2(torch.floor(torch.log2(top.clamp(min=1e-300))))
    # the logarithm may land on the wrong side of a power of two
    below = torch.where(below > top, below / 2, torch.where(below * 2 <= top, below * 2, below))
    step = range15 / 15
    step = torch.where(step > below * 2.0 ** -16, step, below * 2.0 ** -16)
    step = _exact_bf16(torch.where(step > 2.0 ** -40, step, torch.full_like(step, 2.0 ** -40)))
    code = _nearest((y - bias) / step)
    code = torch.where(code < 0, torch.zeros_like(code), torch.where(code > 15, torch.full_like(code, 15.0), code))
    z = code * step + bias
    z[flip] = -z[flip]
    return z.flatten(-2)


def exact(case, seed):
    if case["op"] == "write":
        k, v = _rows(case, seed)
        return {"k": _exact_values(k, case["offset"]), "v": _exact_values(v, case["offset"])}
    q, rows_of, lens = _sequences(case, seed)
    pages, heads, hd = case.get("pages", "u4"), case["kv_heads"], case["hd"]
    outs, new = [], {"k": [], "v": []}
    for i, n in enumerate(lens):
        k, v = rows_of(i)
        if pages == "u4":
            k, v = _exact_values(k, 0), _exact_values(v, 0)
        elif pages == "bf16":
            k, v = _exact_bf16(k.double()), _exact_bf16(v.double())
        k, v = k.double(), v.double()
        new["k"].append(k[-1])
        new["v"].append(v[-1])
        sinks, start = _visible(case, n)
        rows = torch.cat([torch.arange(sinks), torch.arange(start, n)]).cuda()
        qi = q[i].double().view(heads, -1, hd)
        s = torch.einsum("hgd,rhd->hgr", qi, k[rows]) / math.sqrt(hd)
        p = torch.softmax(s, -1)
        outs.append(torch.einsum("hgr,rhd->hgd", p, v[rows]).reshape(-1, hd))
    result = {"out": torch.stack(outs)}
    if case.get("append"):
        result.update(new_k=torch.stack(new["k"]), new_v=torch.stack(new["v"]))
    return result
