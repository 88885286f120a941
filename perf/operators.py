"""What the gradient operators are measured on: the norm over many tensors, clipping by it, and the sum over
micro-batches.

A case names a table of gradients (the shapes of a training configuration, or a random split), its types and the
operator.  Gradients lie in one flat buffer, as the framework's arenas and flat gradient buckets hold them; `align` is
the alignment of each tensor in elements (16: the arena layout, 1: packed without gaps, as flat buckets often are, so
that most tensors start off a vector boundary).  What lies between two tensors is zero and belongs to none.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
P = {"l1": 1.0, "l2": 2.0, "max": math.inf}


# -- tables ---------------------------------------------------------------------------------------------------------
def sizes_of(case):
    """Element counts of a case's tensors; they depend on the case alone."""
    kind = case["table"]
    if kind == "gpt2":  # GPT-2 small, the leaves of the framework's own benchmark
        d = 768
        out = [50257 * d, 1024 * d]
        for _ in range(12):
            out += [d, d, d * 3 * d, 3 * d, d * d, d, d, d, d * 4 * d, 4 * d, 4 * d * d, d]
        return out + [d, d]
    if kind == "llama":  # layers of the Llama-3-8B shapes, and the embedding where asked for
        d, kv, ffn = 4096, 1024, 14336
        out = [128256 * d] if case["embedding"] else []
        for _ in range(case["layers"]):
            out += [d * d, d * kv, d * kv, d * d, d * ffn, d * ffn, ffn * d, d, d]
        return out
    if kind == "equal":
        return [case["each"]] * case["tensors"]
    # "random": log-uniform shares of `total`, at least one element each
    r = random.Random(case["shape_seed"])
    share = [math.exp(r.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
    scale = case["total"] / sum(share)
    return [max(1, int(x * scale)) for x in share]


def offsets_of(sizes, align):
    at, out = 0, []
    for n in sizes:
        at = -(-at // align) * align
        out.append(at)
        at += n
    return out, max(1, at)


def listed():
    return [
        # -- the norm
        # one small tensor: what a call costs when there is nothing to read
        dict(name="norm one vector", op="norm", table="equal", tensors=1, each=4097, align=16, g="f32", p="l2",
             each_norm=False),
        # the logged norm of a whole small model, f32 gradients
        dict(name="norm gpt2 f32", op="norm", table="gpt2", align=16, g="f32", p="l2", each_norm=False),
        # a shard of a large model with a norm per tensor for the log, bf16 gradients
        dict(name="norm llama bf16 each", op="norm", table="llama", layers=4, embedding=True, align=16, g="bf16",
             p="l2", each_norm=True),
        # the largest value of f16 gradients under a loss scale, packed buckets of odd sizes
        dict(name="norm ragged f16 max", op="norm", table="random", tensors=257, total=19_000_003, shape_seed=3,
             align=1, g="f16", p="max", each_norm=True),
        # -- clipping
        # the norms' weights of a small model
        dict(name="clip 25 vectors", op="clip", table="equal", tensors=25, each=768, align=16, g="f32", out="f32",
             p="l2", limit="over"),
        # a small model whose norm is over the limit: everything is written
        dict(name="clip gpt2 f32", op="clip", table="gpt2", align=16, g="f32", out="f32", p="l2", limit="over"),
        # the same in place with the norm under the limit, as most steps of a run are: nothing is written
        dict(name="clip gpt2 f32 under", op="clip", table="gpt2", align=16, g="f32", out="same", p="l2",
             limit="under"),
        # f32 sums of a few large layers, clipped into the bf16 gradients that the step reads
        dict(name="clip llama f32 to bf16", op="clip", table="llama", layers=2, embedding=False, align=16, g="f32",
             out="bf16", p="l2", limit="over"),
        # packed bf16 buckets of odd sizes by their L1 norm
        dict(name="clip ragged bf16 l1", op="clip", table="random", tensors=301, total=7_340_033, shape_seed=8,
             align=1, g="bf16", out="bf16", p="l1", limit="over"),
        # -- the sum over micro-batches
        # a few small tensors
        dict(name="sum 12 vectors", op="sum", table="equal", tensors=12, each=2049, align=16, g="bf16", alpha=1.0,
             first=False, p="none"),
        # the last micro-batch of a small model, with the norm of the sum
        dict(name="sum gpt2 bf16 norm", op="sum", table="gpt2", align=16, g="bf16", alpha=0.125, first=False, p="l2"),
        # the first micro-batch of some large layers, f16 gradients under a loss scale
        dict(name="sum llama f16 first", op="sum", table="llama", layers=2, embedding=False, align=16, g="f16",
             alpha=2.0 ** -12, first=True, p="none"),
    ]


def draw(rng):
    """Tables of 1 to 600 tensors and a thousand to four hundred million elements."""
    op = rng.choice(["norm", "clip", "sum"])
    total = int(math.exp(rng.uniform(math.log(1e3), math.log(4e8))))
    tensors = max(1, min(int(math.exp(rng.uniform(0.0, math.log(600)))), total // 4))
    case = dict(op=op, table="random", tensors=tensors, total=total, shape_seed=rng.randrange(1 << 30),
                align=rng.choice([1, 16]), g=rng.choice(["f32", "bf16", "f16"]))
    if op == "norm":
        case.update(p=rng.choice(["l1", "l2", "max"]), each_norm=rng.random() < 0.5)
    elif op == "clip":
        limit = rng.choice(["over", "over", "under"])
        case.update(p=rng.choice(["l1", "l2", "l2", "max"]), limit=limit,
                    out="same" if limit == "under" else rng.choice(["f32", "bf16", case["g"]]))
    else:
        case.update(alpha=rng.choice([1.0, 0.125, 2.0 ** -12]), first=rng.random() < 0.3,
                    p=rng.choice(["none", "l1", "l2", "max"]))
    return case


# -- inputs ---------------------------------------------------------------------------------------------------------
def inputs(case, seed):
    """The gradients, flat and as tensors, and what the call takes beside them."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    sizes = sizes_of(case)
    at, total = offsets_of(sizes, case["align"])
    r = random.Random(seed + 1)
    # f16 gradients come with a loss scale
    unit = 4096.0 if case["g"] == "f16" else 1.0
    flat = torch.zeros(total, dtype=DT[case["g"]], device="cuda")
    grads = [flat[a:a + n] for a, n in zip(at, sizes)]
    expect = {"l1": 0.0, "l2": 0.0, "max": 0.0, "none": 0.0}
    for g in grads:
        std = 10.0 ** r.uniform(-5.0, -2.5) * unit  # tensors of one model differ by orders of magnitude
        g.normal_(0.0, std, generator=gen)
        expect["l1"] += std * g.numel() * math.sqrt(2.0 / math.pi)
        expect["l2"] += std * std * g.numel()
        expect["max"] = max(expect["max"], 3.0 * std)
    expect["l2"] = math.sqrt(expect["l2"])
    s = dict(case=case, sizes=sizes, flat=flat, grads=grads)
    if case["op"] == "clip":
        s["max_norm"] = expect[case["p"]] * (0.25 if case["limit"] == "over" else 8.0)
        s["out"] = flat if case["out"] == "same" else torch.zeros(total, dtype=DT[case["out"]], device="cuda")
    if case["op"] == "sum":
        s["out"] = torch.zeros(total, dtype=torch.float32, device="cuda")
        if not case["first"]:  # what earlier micro-batches left
            for a, g in zip(at, grads):
                s["out"][a:a + g.numel()].normal_(0.0, 1e-3, generator=gen)
    if "out" in s:
        s["outs"] = [s["out"][a:a + n] for a, n in zip(at, sizes)]
    return s


def prepare(case, seed):
    s = inputs(case, seed)
    if own:  # the leaf table, which a program with standing gradient buffers builds once
        from tikun_b200 import GradTable

        s["table"] = GradTable(s["grads"], out=s["outs"] if s.get("out") is not None and s["out"] is not s["flat"]
                               else None)
    return s


# -- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    return run_own(state) if own else run_plain(state)


def run_own(s):
    from tikun_b200 import accumulate_grads_, clip_grad_norm_, grad_norm

    case = s["case"]
    if case["op"] == "norm":
        return grad_norm(s["table"], norm_type=P[case["p"]], per_tensor=case["each_norm"])
    if case["op"] == "clip":
        return clip_grad_norm_(s["table"], s["max_norm"], norm_type=P[case["p"]]), s["out"]
    norm = accumulate_grads_(s["table"], alpha=case["alpha"], overwrite=case["first"],
                             norm_type=None if case["p"] == "none" else P[case["p"]])
    return (s["out"],) if norm is None else (norm, s["out"])


def plain_power(x, p):
    """The sum (or largest) of the values' powers, in 64 bits."""
    if p == "max":
        return x.abs().amax().double()
    return (x * x if p == "l2" else x.abs()).sum(dtype=torch.float64)


def plain_root(power, p):
    return (power.sqrt() if p == "l2" else power).float()


def run_plain(s):
    case = s["case"]
    if case["op"] == "norm":
        p = case["p"]
        if not case["each_norm"]:
            return plain_root(plain_power(s["flat"].float(), p), p)
        power = torch.stack([plain_power(g.float(), p) for g in s["grads"]])
        return plain_root(power.amax() if p == "max" else power.sum(), p), plain_root(power, p)
    if case["op"] == "clip":
        x = s["flat"].float()
        norm = plain_root(plain_power(x, case["p"]), case["p"])
        scale = torch.where(norm > s["max_norm"], s["max_norm"] / (norm + 1e-6), 1.0)
        s["out"].copy_(x * scale)
        return norm, s["out"]
    x = s["flat"].float() * case["alpha"]
    if case["first"]:
        s["out"].copy_(x)
    else:
        s["out"] += x
    if case["p"] == "none":
        return (s["out"],)
    return plain_root(plain_power(s["out"], case["p"]), case["p"]), s["out"]


# -- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact_norms(tensors, p):
    """Norm of each tensor, and of all, from f64 values, a piece of 2^26 elements at a time."""
    each = []
    for t in tensors:
        parts = [torch.linalg.vector_norm(piece.double(), P[p]).item() for piece in t.split(1 << 26)]
        each.append(max(parts) if p == "max" else math.fsum(v ** P[p] for v in parts) ** (1.0 / P[p]))
    whole = max(each) if p == "max" else math.fsum(v ** P[p] for v in each) ** (1.0 / P[p])
    dev = tensors[0].device
    return (torch.tensor(whole, dtype=torch.float64, device=dev),
            torch.tensor(each, dtype=torch.float64, device=dev))


def exact(case, seed):
    s = inputs(case, seed)
    if case["op"] == "norm":
        whole, each = exact_norms(s["grads"], case["p"])
        return (whole, each) if case["each_norm"] else whole
    if case["op"] == "clip":
        norm, _ = exact_norms(s["grads"], case["p"])
        factor = s["max_norm"] / (norm.item() + 1e-6) if norm.item() > s["max_norm"] else 1.0
        return norm, s["flat"].double().mul_(factor)
    total = s["flat"].double().mul_(case["alpha"])
    if not case["first"]:
        total += s["out"]
    if case["p"] == "none":
        return (total,)
    at, _ = offsets_of(s["sizes"], case["align"])
    return exact_norms([total[a:a + n] for a, n in zip(at, s["sizes"])], case["p"])[0], total


# -- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    n = sum(sizes_of(case))
    read = n * SIZE[case["g"]]
    if case["op"] == "norm":
        return {"bytes": read + 4 * (1 + (len(sizes_of(case)) if case["each_norm"] else 0)), "flops": 2 * n}
    if case["op"] == "clip":
        if case["limit"] == "under" and case["out"] == "same":  # the gradients stay as they are
            return {"bytes": read + 4, "flops": 2 * n}
        return {"bytes": read + n * (SIZE[case["g"]] if case["out"] == "same" else SIZE[case["out"]]) + 4,
                "flops": 3 * n}
    write = 4 * n if case["first"] else 8 * n
    return {"bytes": read + write, "flops": (2 if case["p"] == "none" else 4) * n}
