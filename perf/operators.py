"""The operators of language models that this library offers, as cases to time and compare.

Rows of an embedding table and their gradient, log probabilities of tokens and their gradient, and the global norm of
many gradients with clipping by it.  With `own` false a case runs in a plain form of elementary torch operations; with
`own` true the same tensors, taken as this library's arrays, go through its own entry points."""
import ctypes
import math

import torch

own = False

IGNORE = -100                     # an id that stands for no token
TYPES = {"float32": (torch.float32, 4), "float16": (torch.float16, 2), "bfloat16": (torch.bfloat16, 2)}
LARGEST = 1.3e9                   # bytes of the largest listed case, by work()


def listed():
    return [
        # one decoding step of a few sequences: latency
        dict(name="embed step", op="embed", n=7, v=50257, d=1024, table="float32", out="float32", ids="int64", pad=0.0, scale=1.0),
        # the tokens of a training batch or of long prompts, with the scaling some models apply
        dict(name="embed batch", op="embed", n=16384, v=50257, d=1024, table="bfloat16", out="bfloat16", ids="int64", pad=0.05, scale=32.0),
        # a small model's or a test's gradient
        dict(name="embed_grad small", op="embed_grad", n=96, v=1000, d=257, dout="float32", grad="float32", ids="int64", pad=0.0,
             scale=1.0, accumulate=False),
        # the dense gradient of one training step, in the type of the main weights
        dict(name="embed_grad batch", op="embed_grad", n=8192, v=50257, d=1024, dout="bfloat16", grad="float32", ids="int64", pad=0.1,
             scale=32.0, accumulate=False),
        # a large batch added to what the output layer left there (tied weights, or one micro-batch of several)
        dict(name="embed_grad accumulate", op="embed_grad", n=65536, v=65536, d=2048, dout="bfloat16", grad="float32", ids="int32", pad=0.3,
             scale=1.0, accumulate=True),
        # decoding under a mask of allowed tokens, one idle slot, with alternatives and entropy: latency
        dict(name="logprobs step", op="logprobs", t=8, v=50257, pitch=50257, type="float32", top=20, entropy=True, mask=0.3, pad=0.0, scale=0.7),
        # scoring long texts, rows off the 16-byte boundaries
        dict(name="logprobs score", op="logprobs", t=4096, v=50257, pitch=50257, type="bfloat16", top=0, entropy=True, mask=0.0, pad=0.1, scale=1.0),
        # many short rows with alternatives
        dict(name="logprobs rows of 1000", op="logprobs", t=65536, v=1000, pitch=1000, type="float32", top=5, entropy=False, mask=0.0, pad=0.0,
             scale=1.0),
        # the gradient of a small test
        dict(name="logprobs_grad small", op="logprobs_grad", t=16, v=1000, pitch=1000, type="float32", entropy=False, mask=0.0, pad=0.0, scale=1.0),
        # the gradient of a policy step: log probabilities and entropy, sequences padded at their ends
        dict(name="logprobs_grad batch", op="logprobs_grad", t=4096, v=50257, pitch=50304, type="bfloat16", entropy=True, mask=0.0, pad=0.1,
             scale=1.0),
        # the gradients of a small model: latency
        dict(name="clip small", op="clip", tensors=12, elements=40007, type="float32", ratio=3.7),
        # the gradients of a model of a few hundred million weights, clipped into the optimiser's copy
        dict(name="clip large", op="clip", tensors=148, elements=300000017, type="bfloat16", ratio=3.7),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["embed", "embed_grad", "logprobs", "logprobs_grad", "clip"])
        any_type = lambda: rng.choice(sorted(TYPES))  # noqa: E731
        pad = rng.choice([0.0, 0.05, 0.3])
        if op == "embed":
            c = dict(op=op, n=_log_int(rng, 1, 65536), v=_log_int(rng, 200, 200000), d=_log_int(rng, 16, 8192), table=any_type(), out=any_type(),
                     ids=rng.choice(["int32", "int64"]), pad=pad, scale=rng.choice([1.0, 22.5]))
        elif op == "embed_grad":
            c = dict(op=op, n=_log_int(rng, 1, 131072), v=_log_int(rng, 200, 200000), d=_log_int(rng, 16, 8192), dout=any_type(), grad=any_type(),
                     ids=rng.choice(["int32", "int64"]), pad=pad, scale=rng.choice([1.0, 22.5]), accumulate=False)
            if c["grad"] == "float32":            # sums over several calls are kept in 32 bits
                c["accumulate"] = rng.random() < 0.5
        elif op in ("logprobs", "logprobs_grad"):
            v = _log_int(rng, 100, 260000)
            c = dict(op=op, t=_log_int(rng, 1, 65536), v=v, pitch=v + rng.choice([0, 0, 1, 47]), type=any_type(), entropy=rng.random() < 0.5,
                     mask=rng.choice([0.0, 0.0, 0.5]), pad=pad, scale=rng.choice([1.0, 0.7, 1.4]))
            if op == "logprobs":
                c["top"] = rng.choice([0, 0, 1, 5, 20, 50])
        else:
            c = dict(op=op, tensors=rng.randint(1, 400), elements=_log_int(rng, 2000, 300000000), type=any_type(), ratio=rng.choice([0.5, 3.7]))
        if work(c)["bytes"] <= LARGEST:
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------

def _ids(case, n, g):
    """Token ids as text has them, a few very often and most hardly ever; a share of them stands for no token."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(case["v"])).long() - 1).clamp_(0, case["v"] - 1) * 7919 % case["v"]
    ids[torch.rand(n, generator=g, device="cuda") < case["pad"]] = IGNORE
    return ids.to(torch.int32 if case.get("ids") == "int32" else torch.int64)


def _cuts(case, seed):
    """Where the tensors of a flat buffer begin and end: sizes of all orders of magnitude, as a model's are."""
    n, k = case["elements"], case["tensors"]
    g = torch.Generator().manual_seed(seed)
    part = torch.exp(6 * torch.rand(k, generator=g, dtype=torch.float64))
    cuts = (torch.cumsum(part, 0) / part.sum() * n).long().tolist()
    return [0] + cuts[:-1] + [n]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def normal(shape, kind, by=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * by).to(TYPES[kind][0])

    s = {"case": case}
    if op == "embed":
        s["table"] = normal((case["v"], case["d"]), case["table"], 0.02)
        s["ids"] = _ids(case, case["n"], g)
        s["out"] = torch.empty((case["n"], case["d"]), device="cuda", dtype=TYPES[case["out"]][0])
    elif op == "embed_grad":
        s["ids"] = _ids(case, case["n"], g)
        s["dout"] = normal((case["n"], case["d"]), case["dout"], 0.01)
        s["grad"] = normal((case["v"], case["d"]), case["grad"], 0.01) if case["accumulate"] else \
            torch.empty((case["v"], case["d"]), device="cuda", dtype=TYPES[case["grad"]][0])
    elif op in ("logprobs", "logprobs_grad"):
        t, v = case["t"], case["v"]
        rows = torch.empty((t, case["pitch"]), device="cuda", dtype=TYPES[case["type"]][0])
        x = rows[:, :v]
        x.copy_(torch.randn((t, v), generator=g, device="cuda").mul_(2.0))
        if case["mask"]:
            x.masked_fill_(torch.rand((t, v), generator=g, device="cuda") < case["mask"], -math.inf)
            if t > 1:
                x[t // 2] = -math.inf          # an idle slot: nothing is allowed
        s["logits"], s["ids"] = x, _ids(case, t, g)
        f32 = dict(device="cuda", dtype=torch.float32)
        if op == "logprobs":
            s["logp"], s["stats"] = torch.empty(t, **f32), torch.empty((t, 2), **f32)
            if case["entropy"]:
                s["entropy"] = torch.empty(t, **f32)
            if case["top"]:
                s["top_logp"] = torch.empty((t, case["top"]), **f32)
                s["top_ids"] = torch.empty((t, case["top"]), device="cuda", dtype=torch.int64)
        else:
            # what the forward pass left, in the type it leaves it in
            s["stats"], s["entropy"] = torch.empty((t, 2), **f32), torch.empty(t, **f32)
            for a in range(0, t, 1024):
                m, ls, z, e = _softmax(x[a:a + 1024].float(), case["scale"])
                s["stats"][a:a + 1024] = torch.cat([m, ls], 1)
                s["entropy"][a:a + 1024] = _entropy(ls, z, e)
            s["dlogp"] = torch.randn(t, generator=g, **f32)
            s["dentropy"] = torch.randn(t, generator=g, **f32) * 0.1
            s["dlogits"] = torch.empty((t, v), device="cuda", dtype=TYPES[case["type"]][0])
    else:
        s["flat"] = normal((case["elements"],), case["type"], 1e-3)
        s["clipped"] = torch.empty_like(s["flat"])
        s["norm"] = torch.empty((), device="cuda", dtype=torch.float32)
        s["max_norm"] = 1e-3 * math.sqrt(case["elements"]) / case["ratio"]
    if own:
        _arrays(s, seed)
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------

def _softmax(x, scale):
    """Largest value of each row, logarithm of the sum of exp(scale * (x - largest)), the exponents and their exp."""
    m = x.amax(1, keepdim=True)
    z = (x - torch.where(torch.isinf(m), torch.zeros_like(m), m)) * scale
    e = torch.exp(z)
    return m, torch.log(e.sum(1, keepdim=True)), z, e


def _entropy(ls, z, e):
    ez = torch.where(e > 0, e * z, torch.zeros_like(e)).sum(1)
    return torch.where(torch.isinf(ls[:, 0]), torch.zeros_like(ez), ls[:, 0] - ez / e.sum(1))


def _order(x):
    """Whole numbers in the order of the values of a row; of equal values the one with the lower index is the larger."""
    b = x.view(torch.int32).long()
    b = torch.where(b < 0, -(b & 0x7fffffff), b)          # -0.0 is equal to 0.0
    return (b << 32) + (0xffffffff - torch.arange(x.shape[1], device=x.device))


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "embed":
        ids = s["ids"].long()
        rows = s["table"][ids.clamp(min=0)].float() * case["scale"]
        return {"out": torch.where((ids == IGNORE)[:, None], torch.zeros_like(rows), rows).to(s["out"].dtype)}
    if op == "embed_grad":
        ids = s["ids"].long()
        sums = torch.zeros((case["v"] + 1, case["d"]), device="cuda")
        sums.index_add_(0, torch.where(ids == IGNORE, torch.full_like(ids, case["v"]), ids), s["dout"].float())
        got = sums[:-1] * case["scale"]
        if case["accumulate"]:
            s["grad"] += got
            return {"grad": s["grad"]}
        return {"grad": got.to(s["grad"].dtype)}
    if op == "clip":
        norm = torch.sqrt(s["flat"].double().square().sum())
        by = torch.where(torch.isfinite(norm) & (norm > s["max_norm"]), s["max_norm"] / norm, torch.ones_like(norm)).float()
        return {"clipped": (s["flat"].float() * by).to(s["flat"].dtype), "norm": norm.float()}
    x, ids, scale = s["logits"].float(), s["ids"], case["scale"]
    at = ids.clamp(min=0)[:, None]
    left_out = ids == IGNORE
    if op == "logprobs":
        m, ls, z, e = _softmax(x, scale)
        nothing = torch.isinf(ls[:, 0])
        logp = torch.where(nothing, torch.full_like(m[:, 0], -math.inf), z.gather(1, at)[:, 0] - ls[:, 0])
        out = {"logp": torch.where(left_out, torch.zeros_like(logp), logp), "stats": torch.cat([m, ls], 1)}
        if case["entropy"]:
            out["entropy"] = _entropy(ls, z, e)
        if case["top"]:
            best = torch.topk(_order(x), case["top"], dim=1).values
            out["top_ids"] = 0xffffffff - (best & 0xffffffff)
            top = z.gather(1, out["top_ids"]) - ls
            out["top_logp"] = torch.where(nothing[:, None], torch.full_like(top, -math.inf), top)
        return out
    m, ls = s["stats"][:, :1], s["stats"][:, 1:]
    nothing = torch.isinf(ls)
    logp = (x - torch.where(nothing, torch.zeros_like(m), m)) * scale - torch.where(nothing, torch.zeros_like(ls), ls)
    p = torch.exp(logp)
    by = torch.where(left_out, torch.zeros_like(s["dlogp"]), s["dlogp"])[:, None]
    d = -by * p
    if case["entropy"]:
        d -= s["dentropy"][:, None] * p * torch.where(p > 0, logp + s["entropy"][:, None], torch.zeros_like(p))
    d.scatter_add_(1, at, by)
    return {"dlogits": torch.where(nothing, torch.zeros_like(d), d * scale).to(s["dlogits"].dtype)}


# ---- the library's calls ----------------------------------------------------------------------------------------

def _arrays(s, seed):
    """The state's tensors as arrays of this library, over the same memory, and the plan that clipping keeps."""
    import libgpuarray_amd as ga
    ctx = ga.get_default_context()
    if ctx is None:
        ctx = ga.init("hip0")
        ga.set_default_context(ctx)
    make = ga._lib.extension("hip_make_buf", ctypes.c_void_p, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t])
    kinds = {torch.bfloat16: ga.bfloat16, torch.float16: "float16", torch.float32: "float32", torch.int32: "int32", torch.int64: "int64"}

    def wrap(x):
        n = (1 + sum((d - 1) * st for d, st in zip(x.shape, x.stride()))) * x.element_size()
        data = make(ctx.ctx, x.data_ptr(), n)
        a = ga.from_gpudata(data, 0, kinds[x.dtype], tuple(x.shape), context=ctx, strides=[st * x.element_size() for st in x.stride()] or None)
        ga._lib.lib.gpudata_release(data)
        return a

    s["ga"] = {k: wrap(x) for k, x in s.items() if isinstance(x, torch.Tensor)}
    if s["case"]["op"] == "clip":
        cuts = _cuts(s["case"], seed)
        flat, clipped = ([s["ga"][k][a:b] for a, b in zip(cuts, cuts[1:])] for k in ("flat", "clipped"))
        s["plan"] = ga.GlobalNorm(flat, out=clipped)
    if s["case"]["op"] == "logprobs":
        s["result"] = ga.TokenLogprobs(*(s["ga"].get(k) for k in ("logp", "entropy", "stats", "top_logp", "top_ids")))
    torch.cuda.synchronize()       # the tensors were made on torch's stream, the calls go to the context's
    s["lib"] = ga


def _call(s):
    case, a, ga = s["case"], s["ga"], s["lib"]
    op = case["op"]
    if op == "embed":
        ga.embedding(a["table"], a["ids"], scale=case["scale"], ignore=IGNORE, out=a["out"], check=False)
        return {"out": s["out"]}
    if op == "embed_grad":
        ga.embedding_grad(a["dout"], a["ids"], a["grad"], scale=case["scale"], ignore=IGNORE, accumulate=case["accumulate"], check=False)
        return {"grad": s["grad"]}
    if op == "clip":
        s["plan"].clip(s["max_norm"], norm=a["norm"])
        return {"clipped": s["clipped"], "norm": s["norm"]}
    if op == "logprobs":
        ga.token_logprobs(a["logits"], a["ids"], scale=case["scale"], ignore=IGNORE, out=s["result"], check=False)
        return {k: s[k] for k in ("logp", "stats", "entropy", "top_ids", "top_logp") if k in s}
    ga.token_logprobs_grad(a["logits"], a["ids"], a["stats"], a["dlogp"], entropy=a["entropy"] if case["entropy"] else None,
                           dentropy=a["dentropy"] if case["entropy"] else None, scale=case["scale"], ignore=IGNORE, out=a["dlogits"], check=False)
    return {"dlogits": s["dlogits"]}


def run(state):
    return _call(state) if own else _plain(state)


# ---- what a pass cannot do without, and its exact outputs --------------------------------------------------------

def work(case):
    op = case["op"]
    size = lambda k: TYPES[case[k]][1]  # noqa: E731
    if op == "embed":
        id_bytes = 4 if case["ids"] == "int32" else 8
        return {"bytes": case["n"] * (id_bytes + case["d"] * size("out")) + min(case["n"], case["v"]) * case["d"] * size("table"),
                "flops": case["n"] * case["d"]}
    if op == "embed_grad":
        id_bytes = 4 if case["ids"] == "int32" else 8
        table = 2 * min(case["n"], case["v"]) if case["accumulate"] else case["v"]
        return {"bytes": case["n"] * (id_bytes + case["d"] * size("dout")) + table * case["d"] * size("grad"), "flops": 2 * case["n"] * case["d"]}
    if op == "clip":
        return {"bytes": 2 * case["elements"] * size("type"), "flops": 3 * case["elements"]}
    cells = case["t"] * case["v"]
    if op == "logprobs":
        return {"bytes": cells * size("type") + case["t"] * (8 + 16 + 12 * case["top"]), "flops": (6 if case["entropy"] else 4) * cells}
    return {"bytes": 2 * cells * size("type") + case["t"] * 28, "flops": (8 if case["entropy"] else 5) * cells}


def exact(case, seed):
    """The outputs in 64 bits, from the definitions: softmax by rows, sums over equal ids, the 2-norm of all elements."""
    s = prepare(case, seed)
    op, f64 = case["op"], torch.float64
    if op == "embed":
        keep = (s["ids"] != IGNORE).to(f64)
        return {"out": torch.nn.functional.embedding(s["ids"].long().clamp(min=0), s["table"].to(f64)) * case["scale"] * keep[:, None]}
    if op == "embed_grad":
        keep = (s["ids"] != IGNORE).nonzero()[:, 0]
        total = s["grad"].to(f64) if case["accumulate"] else torch.zeros(s["grad"].shape, device="cuda", dtype=f64)
        total.index_put_((s["ids"][keep].long(),), s["dout"][keep].to(f64) * case["scale"], accumulate=True)
        return {"grad": total}
    if op == "clip":
        x = s["flat"].to(f64)
        norm = torch.linalg.vector_norm(x)
        return {"clipped": x * min(1.0, s["max_norm"] / norm.item()), "norm": norm}
    n, scale, parts = case["t"], case["scale"], []
    for a in range(0, n, 1024):
        x = s["logits"][a:a + 1024].to(f64)
        ids = s["ids"][a:a + 1024].long()
        lse = torch.logsumexp(x * scale, 1)
        there = torch.isfinite(lse)
        logs = x * scale - torch.where(there, lse, torch.zeros_like(lse))[:, None]
        keep = (ids != IGNORE).to(f64)
        p = torch.exp(logs)
        plogp = torch.special.xlogy(p, p)
        if op == "logprobs":
            own_logp = logs[torch.arange(len(ids), device="cuda"), ids.clamp(min=0)]
            top = x.max(1).values
            part = {"logp": torch.where(keep > 0, own_logp, torch.zeros_like(own_logp)),
                    "stats": torch.stack([top, torch.where(there, lse - scale * top, lse)], 1)}
            if case["entropy"]:
                part["entropy"] = -plogp.sum(1)
            if case["top"]:
                part["top_logp"] = torch.sort(logs, dim=1, descending=True).values[:, :case["top"]]
        else:
            hot = torch.nn.functional.one_hot(ids.clamp(min=0), case["v"])
            grad = (s["dlogp"][a:a + 1024].to(f64) * keep)[:, None] * (hot - p)
            if case["entropy"]:
                h = -plogp.sum(1, keepdim=True)
                grad -= s["dentropy"][a:a + 1024].to(f64)[:, None] * (plogp + p * h)
            part = {"dlogits": (grad * scale) * there[:, None]}
        parts.append(part)
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if case.get("top"):
        out["top_ids"] = None
    return out
