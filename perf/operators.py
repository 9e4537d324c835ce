"""What is measured of the operators over rows of scores: a row holds one score (logit) per entry of a vocabulary.

  top      the k largest scores of every row in falling order, their indices and the row's log-sum-exp: what a
           teacher model hands over for distillation
  sample   one index per row drawn by temperature, top-k, top-p and min-p from a given random number: how a model
           answers
  loss     Kullback-Leibler divergence of a student's rows from a teacher's top scores (forward)
  back     its gradient from the statistics of the forward pass and an upstream gradient per row (backward)
  train    loss and gradient in one call, as a training step makes it

``run`` computes the plain form with elementary torch operations, or makes the library's own calls when ``own`` is
set.  ``exact`` computes the same from the definitions in 64 bits, block by block.
"""
import importlib
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}

_context = []


def listed():
    return [
        # one request answered on its own: the latency of a single token with the usual settings
        dict(name="sample-one", op="sample", rows=1, vocab=32768, pitch=32768, type="bf16", temperature=0.8, top_k=50,
             top_p=0.95, min_p=0.0, mixed=False, allowed=False),
        # a serving batch where every request has settings of its own, greedy ones among them; odd vocabulary
        dict(name="sample-mixed", op="sample", rows=64, vocab=100003, pitch=100003, type="bf16", temperature=1.0, top_k=0,
             top_p=1.0, min_p=0.0, mixed=True, allowed=False),
        # a batch of answers held to a grammar: a bit per entry says what may follow, 32-bit scores
        dict(name="sample-allowed", op="sample", rows=48, vocab=50257, pitch=50304, type="f32", temperature=0.7, top_k=0,
             top_p=0.9, min_p=0.02, mixed=False, allowed=True),
        # rollouts for reinforcement learning: many rows, nothing cut off, so every entry counts
        dict(name="sample-rollouts", op="sample", rows=1024, vocab=131072, pitch=131072, type="bf16", temperature=1.0, top_k=0,
             top_p=1.0, min_p=0.0, mixed=False, allowed=False),
        # a few positions of a teacher, many scores kept, 32-bit
        dict(name="top-few", op="top", rows=24, vocab=50257, pitch=50304, type="f32", k=512, tau=1.0),
        # a teacher's pass over a batch of documents: the scores that are stored for the student
        dict(name="top-many", op="top", rows=2048, vocab=131072, pitch=131072, type="bf16", k=64, tau=2.0),
        # the loss alone, as an evaluation takes it; scores renormalised over what was kept
        dict(name="loss-eval", op="loss", rows=2048, vocab=50257, pitch=50257, type="f32", k=32, tau=1.0, rest=False, masked=100),
        # the loss of a short batch
        dict(name="loss-short", op="loss", rows=48, vocab=32768, pitch=32768, type="bf16", k=20, tau=1.0, rest=True, masked=5),
        # the backward pass of a program that runs forward and backward apart, odd vocabulary
        dict(name="back-odd", op="back", rows=1500, vocab=100003, pitch=100003, type="f16", k=100, tau=2.0, rest=True, masked=77),
        # the backward pass of a short batch, 32-bit
        dict(name="back-short", op="back", rows=32, vocab=32768, pitch=32768, type="f32", k=16, tau=1.0, rest=False, masked=3),
        # a training step over a packed batch, what the kept scores leave out counted as one more entry
        dict(name="train-packed", op="train", rows=4096, vocab=131072, pitch=131072, type="bf16", k=64, tau=1.0, rest=True, masked=256),
        # a training step of a small model, padded rows
        dict(name="train-small", op="train", rows=512, vocab=32001, pitch=32064, type="bf16", k=8, tau=1.5, rest=False, masked=64),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "top", "loss", "back", "train"])
    vocab = _log_uniform(rng, 1000, 160000)
    if rng.random() < 0.5:
        vocab = max(1024, vocab // 64 * 64)
    kind = rng.choice(["f32", "f16", "bf16", "bf16"])
    most = {"sample": 100e6, "top": 200e6}.get(op, 400e6)
    rows = _log_uniform(rng, 1, max(2, min(8192, int(most / vocab))))
    pitch = rng.choice([vocab, (vocab + 63) // 64 * 64])
    case = dict(op=op, rows=rows, vocab=vocab, pitch=pitch, type=kind)
    if op == "sample":
        case.update(temperature=round(rng.uniform(0.3, 1.5), 3), top_k=rng.choice([0, 0, 1, 10, 50, 200, 1000]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]), min_p=rng.choice([0.0, round(rng.uniform(0.01, 0.2), 3)]),
                    mixed=rng.random() < 0.4, allowed=rng.random() < 0.3)
    else:
        case.update(k=min(_log_uniform(rng, 1, 1024), vocab), tau=rng.choice([1.0, round(rng.uniform(0.5, 4.0), 2)]))
        if op != "top":
            case.update(rest=rng.random() < 0.5, masked=rng.choice([0, rows // 7]))
    return case


# ------------------------------------------------------------------ inputs
def _rows(buffer, rows, vocab, pitch):
    return buffer.as_strided((rows, vocab), (pitch, 1))


def _scores(gen, rows, vocab, pitch, kind):
    """Scores as a language model gives them: a broad bulk and, in every row, some entries that stand out, by more
    in rows where the model is sure; the last entries of the vocabulary are padding and hold -inf."""
    x = torch.empty(rows * pitch, dtype=TYPES[kind], device="cuda")
    v = _rows(x, rows, vocab, pitch)
    v.normal_(0.0, 1.0, generator=gen).mul_(2.0)
    n = min(64, vocab)
    part = vocab // n  # one entry out of each part of the vocabulary, so that no two are the same
    where = torch.randint(0, part, (rows, n), generator=gen, device="cuda") + torch.arange(n, device="cuda") * part
    where = where.gather(1, torch.rand(rows, n, generator=gen, device="cuda").argsort(1))
    sure = torch.rand(rows, 1, generator=gen, device="cuda") * 10.0 + 5.0
    falls = 1.0 - torch.log1p(torch.arange(n, device="cuda", dtype=torch.float32)) / math.log(n + 1.0)
    v.scatter_(1, where, (sure * (0.4 + 0.6 * falls)).to(v.dtype))
    v[:, vocab - vocab // 500:] = -math.inf
    return v


def _settings(gen, case):
    n = case["rows"]
    u = torch.rand(n, generator=gen, device="cuda")
    full = lambda value, dtype: torch.full((n,), value, dtype=dtype, device="cuda")  # noqa: E731
    if not case["mixed"]:
        return dict(uniform=u, temperature=full(case["temperature"], torch.float32),
                    top_k=full(case["top_k"], torch.int32) if case["top_k"] > 0 else None,
                    top_p=full(case["top_p"], torch.float32) if case["top_p"] < 1 else None,
                    min_p=full(case["min_p"], torch.float32) if case["min_p"] > 0 else None)
    pick = lambda values, dtype: torch.tensor(values, dtype=dtype, device="cuda")[  # noqa: E731
        torch.randint(0, len(values), (n,), generator=gen, device="cuda")]
    return dict(uniform=u, temperature=pick([0.0, 0.2, 0.7, 0.7, 1.0, 1.0, 1.3], torch.float32),
                top_k=pick([0, 0, 1, 20, 50, 50, 400], torch.int32), top_p=pick([1.0, 1.0, 0.5, 0.9, 0.95], torch.float32),
                min_p=pick([0.0, 0.0, 0.0, 0.05, 0.1], torch.float32))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab, pitch, kind = case["rows"], case["vocab"], case["pitch"], case["type"]
    x = _scores(gen, rows, vocab, pitch, kind)
    empty = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    s = dict(op=case["op"], x=x)
    if case["op"] == "sample":
        s.update(_settings(gen, case), token=empty(rows, torch.int32), logprob=empty(rows, torch.float32), allowed=None)
        if case["allowed"]:
            words = (vocab + 31) // 32
            bits = lambda: torch.randint(-2**31, 2**31, (rows, words), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)  # noqa: E731
            s["allowed"] = bits() & bits()
            s["allowed"][rows // 2:] |= bits()[rows // 2:]
            if rows > 2:
                s["allowed"][rows - 1] = 0  # a row that may not go on
                x[rows - 1, : vocab // 2] = math.nan
                x[0].masked_fill_(~_bits(s["allowed"][:1], vocab)[0], math.inf)
        return s
    k = case["k"]
    s.update(tau=case["tau"])
    if case["op"] == "top":
        s.update(k=k, values=empty((rows, k), x.dtype), index=empty((rows, k), torch.int32), lse=empty(rows, torch.float32))
        return s
    # the teacher agrees with the student up to noise; its rows are made in blocks to stay small
    values, index, lse = empty((rows, k), x.dtype), empty((rows, k), torch.int32), empty(rows, torch.float32)
    stats = empty((rows, 4), torch.float32)
    # a mean over the rows; gradients in 16-bit floats with 5 exponent bits are scaled up, as such training does
    weight = torch.full((rows,), (16384.0 if kind == "f16" else 1.0) / rows, device="cuda")
    weight[rows - case["masked"]:] = 0.0
    for r in range(0, rows, 512):
        t = x[r:r + 512].float()
        t += torch.randn(t.shape, generator=gen, device="cuda").mul_(0.7)
        top = t.topk(k, dim=1)
        values[r:r + 512], index[r:r + 512] = top.values.to(x.dtype), top.indices.to(torch.int32)
        lse[r:r + 512] = torch.logsumexp(t.mul_(1.0 / case["tau"]), 1)
    if k > 4:  # a teacher that kept fewer entries for some rows
        index[::5, k - 2:] = -1
    s.update(values=values, index=index, weight=weight, teacher_lse=lse if case["rest"] else None, stats=stats)
    if case["masked"]:
        x[rows - case["masked"]:, ::3] = math.nan  # rows that do not count hold whatever was there
    if case["op"] == "back":
        s["upstream"] = torch.rand(rows, generator=gen, device="cuda") + 0.5
        for r in range(0, rows, 512):
            part = slice(r, r + 512)
            stats[part] = _statistics(x[part], values[part], index[part], s["teacher_lse"][part] if case["rest"] else None, weight[part], case["tau"])
    if case["op"] != "loss":
        s["grad"] = _rows(empty(rows * pitch, x.dtype), rows, vocab, pitch)
    if case["op"] != "back":
        s["loss"] = empty(rows, torch.float32)
    return s


# -------------------------------------------------------------- plain forms
def _bits(words, vocab):
    """bool [rows, vocab] from 32-bit words, bit j % 32 of word j / 32."""
    shift = torch.arange(32, device=words.device, dtype=torch.int32)
    return ((words[:, :, None] >> shift) & 1).bool().flatten(1)[:, :vocab]


def _top(x, k, tau):
    z = x.float()
    z = torch.where(torch.isnan(z), -math.inf, z)
    # one whole number per entry that orders by score and then by the lower index, so that ties are settled
    bits = (z + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    order = order * 2**32 + (2**31 - torch.arange(x.shape[1], device=x.device))
    at = order.topk(k, dim=1).indices
    value = z.gather(1, at)
    m = z.amax(1, keepdim=True)
    e = torch.exp((z - torch.where(m > -math.inf, m, 0.0)) / tau)
    lse = m[:, 0] / tau + torch.log(e.sum(1))
    lse = torch.where(m[:, 0] > -math.inf, lse, -math.inf)
    return value.to(x.dtype), torch.where(value > -math.inf, at, -1).to(torch.int32), lse


def _sample(x, uniform, temperature, top_k, top_p, min_p, allowed):
    # 64 bits: a sum next to a border decides between two indices
    z = x.double()
    z = torch.where(torch.isnan(z), -math.inf, z)
    if allowed is not None:
        z = torch.where(_bits(allowed, x.shape[1]), z, -math.inf)
    warm = (temperature > 0)[:, None]
    m = z.amax(1, keepdim=True)
    w = torch.exp((z - m) / torch.where(warm, temperature[:, None], 1.0).double())
    w = torch.where(z == m, 1.0, torch.where(z > -math.inf, w, 0.0))
    w, at = torch.where(m > -math.inf, w, 0.0), torch.sort(z, dim=1, descending=True, stable=True).indices
    sorted_w = w.gather(1, at)
    rank = torch.arange(x.shape[1], device=x.device)[None, :]
    keep = warm | (rank < 1)
    if top_k is not None:
        keep = keep & ((rank < top_k[:, None]) | (top_k[:, None] <= 0))
    if top_p is not None:
        reach = torch.cumsum(torch.where(keep, sorted_w, 0.0), 1)
        limit = top_p[:, None].double() * reach[:, -1:]
        keep = keep & ((reach - sorted_w < limit) | (rank < 1) | ~(top_p[:, None] < 1))
    if min_p is not None:
        keep = keep & ((sorted_w >= min_p[:, None].double().clamp(max=1.0)) | ~(min_p[:, None] > 0))
    w = torch.where(torch.zeros_like(keep).scatter(1, at, keep), w, 0.0)
    reach = torch.cumsum(w, 1)
    total = reach[:, -1:]
    token = (reach <= uniform[:, None].double() * total).sum(1, keepdim=True)
    last = (x.shape[1] - 1 - torch.argmax((w > 0).flip(1).int(), dim=1, keepdim=True))
    token = torch.minimum(token, last)
    none = total[:, 0] <= 0
    logprob = torch.where(none, -math.inf, torch.log(w.gather(1, token) / total)[:, 0])
    return torch.where(none, -1, token[:, 0]).to(torch.int32), logprob.float()


def _teacher(z, values, index, teacher_lse, tau):
    """Valid entries, their indices and log-probabilities (64 bits: rows x k is small), and the mass of the rest."""
    valid = (index >= 0) & (index < z.shape[1]) & (values > -math.inf)
    t = torch.where(valid, values.double() / tau, -math.inf)
    if teacher_lse is None:
        top = t.amax(1, keepdim=True)
        top = torch.where(top > -math.inf, top, 0.0)
        norm = top + torch.log(torch.exp(t - top).sum(1, keepdim=True))
    else:
        norm = teacher_lse[:, None].double()
    logp = t - norm
    p = torch.where(valid, torch.exp(logp), 0.0)
    rest = None if teacher_lse is None else (1.0 - p.sum(1)).clamp(min=0.0)
    return valid, torch.where(valid, index, 0).long(), logp, p, rest


def _student(z, valid, index, rest):
    """Row maximum, exp(z - max), its sum, and log of the share of all that the teacher did not name."""
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, dtype=torch.float64)
    if rest is None:
        return m, e, total, None, None
    member = torch.zeros(z.shape[0], z.shape[1] + 1, dtype=torch.bool, device=z.device)
    member = member.scatter_(1, torch.where(valid, index, z.shape[1]), True)[:, :-1]
    others = torch.where(member, -math.inf, z)
    most = others.amax(1, keepdim=True)
    share = torch.exp(others - torch.where(most > -math.inf, most, 0.0)).sum(1, dtype=torch.float64)
    return m, e, total, member, most[:, 0].double() + torch.log(share) - m[:, 0].double() - torch.log(total)


def _coefficients(p, rest, log_share):
    """(factor of the student's probability at the teacher's entries, elsewhere)"""
    if rest is None:
        return p.sum(1), p.sum(1), rest
    rest = torch.where(log_share > -math.inf, rest, 0.0)
    s = p.sum(1) + rest
    return s, torch.where(rest > 0, s - rest * torch.exp(-log_share), s), rest


def _statistics(x, values, index, teacher_lse, weight, tau):
    """What the forward pass keeps for the backward pass: row maximum, 1 / sum, and the two factors."""
    z = x.float() / tau
    valid, index, _, p, rest = _teacher(z, values, index, teacher_lse, tau)
    m, _, total, _, log_share = _student(z, valid, index, rest)
    s, c, _ = _coefficients(p, rest, log_share)
    live = (weight != 0) & valid.any(1) & ~(m[:, 0] == -math.inf)
    stats = torch.stack([x.float().amax(1).double(), 1.0 / total, s, c], 1)
    return torch.where(live[:, None], stats, 0.0).float()


def _loss(x, values, index, teacher_lse, weight, tau, with_gradient):
    z = x.float() / tau
    valid, index, logp, p, rest = _teacher(z, values, index, teacher_lse, tau)
    m, e, total, member, log_share = _student(z, valid, index, rest)
    s, c, rest = _coefficients(p, rest, log_share)
    logq = z.gather(1, index).double() - m.double() - torch.log(total)[:, None]
    loss = torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    if rest is not None:
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - log_share), 0.0)
    live = (weight != 0) & valid.any(1) & ~(m[:, 0] == -math.inf)
    loss = torch.where(live, weight * loss, 0.0).float()
    if not with_gradient:
        return loss
    return loss, _gradient(x.dtype, e, 1.0 / total, s, c, member, p, index, weight / tau, live)


def _gradient(dtype, e, inverse, s, c, member, p, index, g, live):
    factor = (g * c * inverse).float()[:, None]
    if member is not None:
        factor = torch.where(member, (g * s * inverse).float()[:, None], factor)
    d = (e * factor).scatter_add_(1, index, (-g[:, None] * p).float())
    return torch.where(live[:, None], d, 0.0).to(dtype)


def _back(x, values, index, teacher_lse, weight, tau, stats, upstream):
    z = x.float()
    valid, index, _, p, rest = _teacher(z, values, index, teacher_lse, tau)
    e = torch.exp((z - stats[:, :1]) / tau)
    member = None
    if rest is not None:
        member = torch.zeros(z.shape[0], z.shape[1] + 1, dtype=torch.bool, device=z.device)
        member = member.scatter_(1, torch.where(valid, index, z.shape[1]), True)[:, :-1]
    return _gradient(x.dtype, e, stats[:, 1], stats[:, 2], stats[:, 3], member, p, index, upstream * weight / tau, stats[:, 1] != 0)


# --------------------------------------------------------------------- run
def _handle():
    if not _context:
        _context.append(importlib.import_module("accelerate-cuda_b200").Context(torch.cuda.current_device()))
    return _context[0]


def run(s):
    op = s["op"]
    if not own:
        if op == "sample":
            return dict(zip(("token", "logprob"), _sample(s["x"], s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["allowed"])))
        if op == "top":
            return dict(zip(("values", "index", "lse"), _top(s["x"], s["k"], s["tau"])))
        if op == "loss":
            return dict(loss=_loss(s["x"], s["values"], s["index"], s["teacher_lse"], s["weight"], s["tau"], False))
        if op == "train":
            return dict(zip(("loss", "grad"), _loss(s["x"], s["values"], s["index"], s["teacher_lse"], s["weight"], s["tau"], True)))
        return dict(grad=_back(s["x"], s["values"], s["index"], s["teacher_lse"], s["weight"], s["tau"], s["stats"], s["upstream"]))
    ctx = _handle()
    if op == "sample":
        ctx.sample_rows(s["x"], s["uniform"], s["token"], logprob=s["logprob"], temperature=s["temperature"], top_k=s["top_k"],
                        top_p=s["top_p"], min_p=s["min_p"], allowed=s["allowed"])
        return dict(token=s["token"], logprob=s["logprob"])
    if op == "top":
        ctx.top_rows(s["x"], s["values"], s["index"], lse=s["lse"], temperature=s["tau"])
        return dict(values=s["values"], index=s["index"], lse=s["lse"])
    if op == "back":
        ctx.distill_rows_backward(s["x"], s["values"], s["index"], s["stats"], s["upstream"], s["grad"],
                                  teacher_lse=s["teacher_lse"], weight=s["weight"], temperature=s["tau"])
        return dict(grad=s["grad"])
    ctx.distill_rows(s["x"], s["values"], s["index"], s["loss"], grad=s.get("grad"), stats=s["stats"] if op == "loss" else None,
                     teacher_lse=s["teacher_lse"], weight=s["weight"], temperature=s["tau"])
    return dict(loss=s["loss"]) if op == "loss" else dict(loss=s["loss"], grad=s["grad"])


def work(case):
    rows, vocab, size = case["rows"], case["vocab"], BYTES[case["type"]]
    row = vocab * size
    if case["op"] == "sample":
        settings = 4 + 4 + 4 * (3 if case["mixed"] else (case["top_k"] > 0) + (case["top_p"] < 1) + (case["min_p"] > 0))
        mask = (vocab + 31) // 32 * 4 if case["allowed"] else 0
        return dict(bytes=rows * (row + mask + settings + 8), flops=rows * vocab * 4)
    k = case["k"]
    if case["op"] == "top":
        return dict(bytes=rows * (row + k * (size + 4) + 4), flops=rows * vocab * 4)
    live = rows - case["masked"]
    teacher = live * (k * (size + 4) + (4 if case["rest"] else 0)) + rows * 4
    if case["op"] == "loss":
        return dict(bytes=live * row + teacher + rows * 20, flops=live * vocab * 4)
    if case["op"] == "train":
        return dict(bytes=live * row + rows * row + teacher + rows * 4, flops=live * vocab * 6)
    return dict(bytes=live * row + rows * row + teacher + live * 20, flops=live * vocab * 5)


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, a block of rows at a time."""
    s = prepare(case, seed)
    rows, vocab = case["rows"], case["vocab"]
    step = max(1, (1 << 25) // vocab)
    parts = []
    for r in range(0, rows, step):
        cut = {key: v[r:r + step] if torch.is_tensor(v) and v.shape[0] == rows else v for key, v in s.items()}
        parts.append({"sample": _exact_sample, "top": _exact_top}.get(case["op"], _exact_distill)(cut))
    whole = {key: torch.cat([p[key] for p in parts]) for key in parts[0]}
    return {key: whole[key] for key in dict(sample=("token", "logprob"), top=("values", "index", "lse"), loss=("loss",),
                                            back=("grad",), train=("loss", "grad"))[case["op"]]}


def _clean(x):
    return torch.nan_to_num(x.double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)


def _exact_top(s):
    x, k = _clean(s["x"]), s["k"]
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    v, i = v[:, :k], i[:, :k].to(torch.int32)
    return dict(values=v, index=i.masked_fill(v == -math.inf, -1), lse=torch.logsumexp(x / s["tau"], 1))


def _exact_sample(s):
    x = _clean(s["x"])
    if s["allowed"] is not None:
        j = torch.arange(x.shape[1], device=x.device)
        may = torch.bitwise_right_shift(s["allowed"][:, j // 32].long(), j % 32) % 2
        x = x.masked_fill(may == 0, -math.inf)
    t = s["temperature"].double()[:, None]
    greedy = t[:, 0] <= 0
    shifted = torch.where(torch.isinf(x), x, x / t.masked_fill(greedy[:, None], 1.0))
    p = torch.softmax(shifted, 1)  # rows of inputs hold either an inf that is masked, or none
    empty = (x == -math.inf).all(1)
    p = p.masked_fill(empty[:, None], 0.0)
    place = torch.empty(x.shape, dtype=torch.int64, device=x.device)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    place.scatter_(1, order, torch.arange(x.shape[1], device=x.device).expand_as(order).contiguous())
    k = torch.full_like(greedy, x.shape[1], dtype=torch.int64)
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"].long(), k)
    k = k.masked_fill(greedy, 1)
    p = p.masked_fill(place >= k[:, None], 0.0)
    if s["top_p"] is not None:
        lined = torch.zeros_like(p).scatter_(1, place, p)
        before = torch.cumsum(lined, 1).roll(1, 1)
        before[:, 0] = -1.0
        enough = before.gather(1, place) >= s["top_p"].double()[:, None] * p.sum(1, keepdim=True)
        p = p.masked_fill(enough & (s["top_p"] < 1)[:, None] & (place > 0), 0.0)
    if s["min_p"] is not None:
        p = p.masked_fill(p < s["min_p"].double()[:, None] * p.amax(1, keepdim=True), 0.0)
    p = p / p.sum(1, keepdim=True)
    c = torch.cumsum(p, 1)
    token = torch.searchsorted(c, s["uniform"].double()[:, None] * c[:, -1:], right=True).clamp(max=x.shape[1] - 1)
    logprob = torch.log(p.gather(1, token))[:, 0].masked_fill(empty, -math.inf)
    return dict(token=token[:, 0].masked_fill(empty, -1).to(torch.int32), logprob=logprob)


def _exact_distill(s):
    tau, x = s["tau"], s["x"].double()
    n, vocab = x.shape
    logq = torch.log_softmax(x / tau, 1)
    index = s["index"].long()
    valid = index >= 0
    t = (s["values"].double() / tau).masked_fill(~valid, -math.inf)
    full = torch.full((n, vocab + 1), -math.inf, dtype=torch.float64, device=x.device)
    norm = torch.logsumexp(t, 1, keepdim=True) if s["teacher_lse"] is None else s["teacher_lse"].double()[:, None]
    logp = full.scatter_(1, index.masked_fill(~valid, vocab), t - norm)[:, :vocab]  # inputs name no index twice
    p = torch.exp(logp)
    named = p > 0
    loss = torch.where(named, p * (logp - logq), 0.0).sum(1)
    q = torch.exp(logq)
    d = q * p.sum(1, keepdim=True) - p
    if s["teacher_lse"] is not None:
        rest = (1.0 - p.sum(1)).clamp(min=0.0)
        left = torch.logsumexp(logq.masked_fill(named, -math.inf), 1)
        counts = (rest > 0) & (left > -math.inf)
        loss = loss + torch.where(counts, rest * (torch.log(rest) - left), 0.0)
        ratio = torch.where(counts, rest * torch.exp(-left), 0.0)
        d = d + q * torch.where(counts, rest, 0.0)[:, None] - torch.where(named, 0.0, q * ratio[:, None])
    weight = s["weight"].double()
    off = (weight == 0) | ~valid.any(1)
    g = weight / tau * (s["upstream"].double() if s["op"] == "back" else 1.0)
    return dict(loss=(weight * loss).masked_fill(off, 0.0), grad=(d * g[:, None]).masked_fill(off[:, None], 0.0))
