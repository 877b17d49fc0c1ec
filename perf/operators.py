"""What is measured of the head losses: softmax cross entropy and distillation
from a teacher's top logits, both straight from hidden states x [rows, dim]
and the head's weight w [vocab, dim] (bf16), forward alone (scoring tokens)
and forward + backward (training), without keeping the logits.

A case: op "ce" or "distill"; mode "score" (row losses and log-sum-exps) or
"train" (those, and the gradients of x and w for given row gradients); rows,
dim, vocab; masked = the share of rows that is left out; scale = the logits'
factor; for distillation topk entries a row, ragged = rows have fewer of them,
and the temperature.
"""
import math

import torch

own = False

_CE = {"op": "ce", "scale": 1.0, "masked": 0.0, "topk": 0, "ragged": False, "temperature": 1.0}
_KD = {"op": "distill", "scale": 1.0, "masked": 0.0, "topk": 64, "ragged": False, "temperature": 2.0}


def listed():
    return [
        # one generated token's log-probability under the 32,000-word head (768 wide)
        dict(_CE, name="ce score 1 token", mode="score", rows=1, dim=768, vocab=32000),
        # a decode batch under the 151,936-word head (1,024 wide): the weight's bytes count
        dict(_CE, name="ce score 16 tokens", mode="score", rows=16, dim=1024, vocab=151936),
        # perplexity of 16 windows of 256 tokens
        dict(_CE, name="ce score 4096 tokens", mode="score", rows=4096, dim=1024, vocab=151936),
        # one window of 256 tokens, the reference's batch of one
        dict(_CE, name="ce train 256", mode="train", rows=256, dim=768, vocab=32000),
        # fine-tuning: prompts and padding are masked
        dict(_CE, name="ce train masked", mode="train", rows=4096, dim=768, vocab=32000, masked=0.6),
        # sizes that divide nothing, and a scaled head
        dict(_CE, name="ce train odd", mode="train", rows=1531, dim=584, vocab=50257, masked=0.25, scale=0.75),
        # the pre-training step: 16 windows of 256 tokens
        dict(_CE, name="ce train 4096", mode="train", rows=4096, dim=1024, vocab=151936),
        # a wide model
        dict(_CE, name="ce train wide", mode="train", rows=2048, dim=4096, vocab=65536),
        # one token's divergence from a teacher
        dict(_KD, name="distill score 1 token", mode="score", rows=1, dim=768, vocab=32000, topk=32),
        # one window
        dict(_KD, name="distill train 256", mode="train", rows=256, dim=768, vocab=32000),
        # sizes that divide nothing, rows with fewer entries and without any
        dict(_KD, name="distill train odd", mode="train", rows=777, dim=1000, vocab=50257, masked=0.1, topk=17,
             ragged=True, temperature=1.0),
        # the pre-training step with a teacher's 64 best
        dict(_KD, name="distill train 4096", mode="train", rows=4096, dim=1024, vocab=151936),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op, mode = rng.choice(["ce", "distill"]), rng.choice(["score", "train", "train"])
    while True:
        rows, dim, vocab = _log(rng, 1, 8192), 8 * _log(rng, 8, 512), _log(rng, 1000, 152000)
        if rows * vocab * dim <= 4096 * 151936 * 1024 and rows * vocab <= 4096 * 151936:
            break
    case = dict(_CE if op == "ce" else _KD, mode=mode, rows=rows, dim=dim, vocab=vocab,
                masked=rng.choice([0.0, 0.0, 0.3, 0.8]), scale=rng.choice([1.0, 1.0, 0.7]))
    if op == "distill":
        case.update(topk=_log(rng, 1, 128), ragged=rng.random() < 0.5, temperature=rng.choice([1.0, 2.0, 3.5]))
    return case


def _kept(case):
    """Rows that are not left out: fixed by the case, so that work() can count them."""
    return max(1, int(round(case["rows"] * (1.0 - case["masked"]))))


_engine = None


def _handle(case):
    """The program's context, with room for this case's calls."""
    global _engine
    import neural_engine_b200 as ne
    if _engine is None:
        _engine = ne.Engine(ne.ModelConfig(1, 128, 256, 2, 2, 64, 256))
    _engine.head_alloc(case["rows"], case["dim"], case["vocab"], case["topk"])
    return _engine


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, dim, vocab, K = case["rows"], case["dim"], case["vocab"], case["topk"]
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")    # noqa: E731
    # logits of a trained model: a spread of 2.5, and the target's raised by up to 15
    w = (randn(vocab, dim) * (2.5 / math.sqrt(dim))).to(torch.bfloat16)
    target = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    toward = w[target].float()
    toward = toward / toward.norm(dim=1, keepdim=True).clamp_min(1e-6)
    x = (randn(rows, dim) + toward * (6.0 * rand(rows, 1))).to(torch.bfloat16)
    out = torch.randperm(rows, generator=g, device="cuda")[_kept(case):]
    left = torch.zeros(rows, dtype=torch.bool, device="cuda")
    left[out] = True
    s = {"case": case, "x": x, "w": w,
         "grad": (0.5 + rand(rows)) / _kept(case)}   # rows weighted, summing to about one
    if case["op"] == "ce":
        s["target"] = torch.where(left, -100, target).to(torch.int32)
    else:
        # a teacher's best entries, best first; the first is the row's target, the others differ from one another
        step = torch.randint(1, max(2, vocab // (K + 1)), (rows, K), generator=g, device="cuda")
        step[:, 0] = 0
        ids = (target[:, None] + step.cumsum(1)) % vocab
        logit = 18.0 - torch.cumsum(0.4 * rand(rows, K), 1) - 3.0 * rand(rows, 1)
        if case["ragged"]:
            have = torch.randint(1, K + 1, (rows, 1), generator=g, device="cuda")
            ids = torch.where(torch.arange(K, device="cuda")[None, :] < have, ids, -1)
        s["ids"] = torch.where(left[:, None], -1, ids).to(torch.int32).contiguous()
        s["teacher"] = logit.float().contiguous()
    if own:
        s["engine"] = _handle(case)
        s["loss"], s["lse"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        if case["mode"] == "train":
            s["dx"], s["dw"] = torch.empty_like(x), torch.empty_like(w)
    return s


def _run_own(s):
    c, e = s["case"], s["engine"]
    at = lambda name: s[name].data_ptr()  # noqa: E731
    head = dict(x=at("x"), w=at("w"), rows=c["rows"], dim=c["dim"], vocab=c["vocab"], scale=c["scale"])
    if c["op"] == "ce":
        want = dict(target=at("target"))
        fwd, bwd = e.head_ce_fwd, e.head_ce_bwd
    else:
        want = dict(ids=at("ids"), teacher=at("teacher"), topk=c["topk"], temperature=c["temperature"])
        fwd, bwd = e.head_distill_fwd, e.head_distill_bwd
    fwd(**head, **want, loss=at("loss"), lse=at("lse"))
    if c["mode"] == "score":
        return {"loss": s["loss"], "lse": s["lse"]}
    bwd(**head, **want, lse=at("lse"), grad=at("grad"), dx=at("dx"), dw=at("dw"))
    return {"loss": s["loss"], "lse": s["lse"], "dx": s["dx"], "dw": s["dw"]}


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    x, w = s["x"].float(), s["w"].float()
    T = c["temperature"]
    u = (x @ w.t()).mul_(c["scale"] / T)
    top = u.amax(1, keepdim=True)
    lse = (u - top).exp_().sum(1).log_() + top[:, 0]
    if c["op"] == "ce":
        valid = s["target"] >= 0
        ids = s["target"].long().clamp_min(0)[:, None]
        p = valid[:, None].float()
        loss = lse - u.gather(1, ids)[:, 0]
    else:
        entry = s["ids"] >= 0
        valid = entry.any(1)
        ids = s["ids"].long().clamp_min(0)
        y = torch.where(entry, s["teacher"] / T, -math.inf)
        e = torch.where(entry, (y - y.amax(1, keepdim=True)).exp(), 0.0)
        total = e.sum(1, keepdim=True)
        p = torch.where(entry, e / total, 0.0)
        logp = torch.where(entry, y - y.amax(1, keepdim=True) - total.log(), 0.0)
        loss = T * T * (torch.where(entry, p * (logp - u.gather(1, ids)), 0.0).sum(1) + lse)
    out = {"loss": torch.where(valid, loss, 0.0), "lse": torch.where(valid, lse, 0.0)}
    if c["mode"] == "score":
        return out
    d = u.sub_(lse[:, None]).exp_()
    d.scatter_add_(1, ids, -p)
    d *= torch.where(valid, s["grad"] * (T * c["scale"]), 0.0)[:, None]
    out["dx"] = (d @ w).to(torch.bfloat16)
    out["dw"] = (d.t() @ x).to(torch.bfloat16)
    return out


def exact(case, seed):
    """The definition in 64 bits, some rows at a time."""
    s = prepare(case, seed)
    rows, vocab, T, scale = case["rows"], case["vocab"], case["temperature"], case["scale"]
    w = s["w"].double()
    loss, lse = (torch.zeros(rows, dtype=torch.float64, device="cuda") for _ in range(2))
    train = case["mode"] == "train"
    dx = torch.zeros(rows, case["dim"], dtype=torch.float64, device="cuda") if train else None
    dw = torch.zeros_like(w) if train else None
    if case["op"] == "ce":
        keep = torch.nonzero(s["target"] >= 0)[:, 0]
    else:
        keep = torch.nonzero((s["ids"] >= 0).any(1))[:, 0]
    for r in keep.split(max(1, (1 << 27) // vocab)):
        x = s["x"][r].double()
        logp = torch.log_softmax((scale / T) * (x @ w.t()), 1)
        # the targets as a dense distribution over the vocabulary
        want = torch.zeros_like(logp)
        if case["op"] == "ce":
            want[torch.arange(len(r), device="cuda"), s["target"][r].long()] = 1.0
            entropy = 0.0
        else:
            have = s["ids"][r] >= 0
            y = (s["teacher"][r].double() / T).masked_fill(~have, -math.inf).softmax(1)
            entropy = torch.special.xlogy(y, y).sum(1)
            want.scatter_add_(1, s["ids"][r].long().clamp_min(0), y)
        loss[r] = T * T * (entropy - (want * logp).sum(1))
        # log p = u - lse, so any one column gives the row's log-sum-exp
        lse[r] = (scale / T) * (x @ w[0]) - logp[:, 0]
        if train:
            dz = (T * scale) * s["grad"][r].double()[:, None] * (logp.exp() - want)
            dx[r] = dz @ w
            dw += dz.t() @ x
    out = {"loss": loss, "lse": lse}
    if train:
        out.update(dx=dx, dw=dw)
    return out


def work(case):
    rows, dim, vocab = _kept(case), case["dim"], case["vocab"]
    weights, entries = 2 * vocab * dim, rows * (4 if case["op"] == "ce" else 8 * case["topk"])
    read = weights + 2 * rows * dim + entries
    written = 8 * case["rows"]
    flops = 2 * rows * vocab * dim
    if case["mode"] == "train":   # dx and dw: two more products of the same size
        read += 4 * rows
        written += weights + 2 * case["rows"] * dim
        flops *= 3
    return {"bytes": read + written, "flops": flops}
