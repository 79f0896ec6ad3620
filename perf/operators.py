"""Measured cases of the Newton-Schulz operators on caller-owned device matrices.

    orthogonalize   X_0 = U / (|U|_F + eps),  X_{k+1} = a_k X_k + b_k (X_k X_k^T) X_k + c_k (X_k X_k^T)^2 X_k
    muon_step       v <- mu v + g,  u = g + mu v,  p <- p (1 - lr wd) - lr s O(u)  with O(u) the above

A case is a list of matrix shapes ("64x288*3": three of them), the types, the arithmetic and the layout.
Matrices of one shape are kept as one stack so that the plain form runs as batched products.
"""
import math

import torch

own = False  # True: run() calls the framework's operators instead of the plain form

EPS = 1e-7
# coefficients of one step each: the quintic that most Muon programs use, five times; and the schedule that
# starts steeper and settles (minimax polynomials of shrinking intervals, first steps the steepest)
QUINTIC = [(3.4445, -4.7750, 2.0315)] * 5
SCHEDULE = [(8.2051, -22.9014, 16.4607), (4.0664, -2.8612, 0.5184), (3.9096, -2.8234, 0.5250),
            (3.2856, -2.4153, 0.4853), (2.2779, -1.6198, 0.3985)]
COEFFICIENTS = {"quintic": QUINTIC, "schedule": SCHEDULE}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEVICE = "cuda:0"


def _case(name, op, shapes, kind="bf16", mode="f16", layout="rows", coefficients="quintic", lr=2e-4):
    return {"name": name, "op": op, "shapes": shapes, "type": kind, "mode": mode, "layout": layout,
            "coefficients": coefficients, "lr": lr}


def listed():
    return [
        # the two convolution filters of the small CNN, flattened: the smallest call, nothing but latency
        _case("orth conv f32", "orthogonalize", "32x9 64x288", "f32", "f32"),
        # the weights of the 784-256-128-10 MLP
        _case("orth mlp f32", "orthogonalize", "256x784 128x256 10x128", "f32", "f32"),
        # every head of twelve output projections by itself: column blocks of 1024 x 1024 matrices
        _case("orth heads bf16", "orthogonalize", "1024x64*192", "bf16", "f16", "columns"),
        # sides that are no multiple of anything
        _case("orth odd bf16", "orthogonalize", "1000x513 37x1201 511x509", "bf16", "f16", "rows", "schedule"),
        # the matrices of one d = 1024 transformer layer (projections, feed-forward up and down)
        _case("orth layer bf16", "orthogonalize", "1024x1024*4 4096x1024 1024x4096", "bf16"),
        # one wide model's projection by itself, and gradients that a library left transposed, to f32 accuracy
        _case("orth 4096 bf16", "orthogonalize", "4096x4096", "bf16"),
        _case("orth transposed f32", "orthogonalize", "2048x2048 768x2048*2", "f32", "f32", "transposed"),
        # optimizer steps: the MLP and the CNN in f32 ...
        _case("step mlp f32", "muon_step", "256x784 128x256 10x128", "f32", "f32", lr=0.02),
        _case("step cnn f32", "muon_step", "32x9 64x288 128x9216 10x128", "f32", "f32", lr=0.02),
        # ... the twelve-layer d = 768 set's projections in bf16 throughout ...
        _case("step d768 bf16", "muon_step", "768x768*48", "bf16"),
        # ... experts of a sparse layer ...
        _case("step experts bf16", "muon_step", "512x1024*64 1024x512*32", "bf16", "f16", "rows", "schedule"),
        # ... and twelve layers of the d = 1024 set with f32 masters and bf16 gradients: the largest
        _case("step d1024 mixed", "muon_step", "1024x1024*48 4096x1024*12 1024x4096*12", "mixed"),
    ]


def _groups(case):
    """[(count, rows, cols), ...] of the case's text."""
    out = []
    for word in case["shapes"].split():
        shape, _, count = word.partition("*")
        rows, cols = shape.split("x")
        out.append((int(count or 1), int(rows), int(cols)))
    return out


def _flops(case):
    """Products that no form can do without, symmetric ones at half: the Gram on the long side, the short-side
    squares of the polynomial chain, the product with the long side at the end."""
    steps = len(COEFFICIENTS[case["coefficients"]])
    total = 0
    for count, rows, cols in _groups(case):
        n, m = min(rows, cols), max(rows, cols)
        total += count * (3 * n * n * m + (4 * steps - 3) * n ** 3)
    return total


def draw(rng):
    largest = _flops(listed()[-1])
    while True:
        op = rng.choice(["orthogonalize", "muon_step"])
        kind, mode, lr = rng.choice([("bf16", "f16", 2e-4), ("bf16", "f16", 2e-4), ("f32", "f32", 0.02),
                                     ("mixed", "f16", 2e-4) if op == "muon_step" else ("f16", "f16", 2e-4)])
        words = []
        for _ in range(rng.randint(1, 3)):
            sides = [max(1, round(2 ** rng.uniform(3, 12))) for _ in range(2)]
            if rng.random() < 0.4:  # model widths are often round numbers
                sides = [max(8, s // 64 * 64) for s in sides]
            count = 1 if rng.random() < 0.5 else round(2 ** rng.uniform(0, 6))
            words.append("%dx%d" % tuple(sides) + ("*%d" % count if count > 1 else ""))
        case = _case("", op, " ".join(words), kind, mode, rng.choice(["rows", "rows", "columns", "transposed"]),
                     rng.choice(["quintic", "quintic", "schedule"]), lr)
        del case["name"]
        if _flops(case) <= largest / 4 and sum(c * r * k for c, r, k in _groups(case)) <= 1 << 27:
            return case


def _types(case):
    """(parameters or outputs, gradients or inputs, velocity)"""
    if case["type"] == "mixed":
        return torch.float32, torch.bfloat16, torch.float32
    kind = TYPES[case["type"]]
    return kind, kind, kind


def _laid_out(x, layout):
    """The stack [count, rows, cols] with the same values in another memory layout."""
    if layout == "transposed":  # columns contiguous
        return x.mT.contiguous().mT
    if layout == "columns":     # column blocks of one wide row-major matrix
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    return x.contiguous()


def _update_like(gen, count, rows, cols, scale):
    """What gradients and their running sums look like: a few strong directions over a floor of noise."""
    rank = max(1, min(rows, cols) // 16)
    left = torch.randn(count, rows, rank, generator=gen, device=DEVICE)
    right = torch.randn(count, rank, cols, generator=gen, device=DEVICE)
    noise = torch.randn(count, rows, cols, generator=gen, device=DEVICE)
    return scale * (torch.bmm(left, right) / math.sqrt(rank) + 0.3 * noise)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    to, of, vel = _types(case)
    state = {"case": case, "groups": []}
    for count, rows, cols in _groups(case):
        group = {"grad": _laid_out(_update_like(gen, count, rows, cols, 1e-3).to(of), case["layout"])}
        if case["op"] == "muon_step":
            group["param"] = _laid_out((torch.randn(count, rows, cols, generator=gen, device=DEVICE)
                                        / math.sqrt(cols)).to(to), case["layout"])
            group["velocity"] = _laid_out(_update_like(gen, count, rows, cols, 5e-3).to(vel), case["layout"])
            group["scale"] = 0.2 * math.sqrt(max(rows, cols))  # an update of the size that Adam's has
        else:
            group["out"] = _laid_out(torch.zeros(count, rows, cols, dtype=to, device=DEVICE), case["layout"])
        state["groups"].append(group)
    if own:  # the plan that a program keeps, and its tables of the matrices
        import volta_b200 as vb

        shapes = [(r, c) for n, r, c in _groups(case) for _ in range(n)]
        plan = vb.NewtonSchulzPlan(shapes, COEFFICIENTS[case["coefficients"]], eps=EPS,
                                   ns_mode=vb.VB_NS_F16 if case["mode"] == "f16" else vb.VB_NS_F32_TC)
        state["plan"] = plan
        state["tables"] = {key: plan.matrices([m for g in state["groups"] for m in g[key].unbind(0)])
                           for key in state["groups"][0] if key != "scale"}
        state["scales"] = [g["scale"] for g in state["groups"] for _ in range(len(g["grad"]))] \
            if case["op"] == "muon_step" else None
    return state


MOMENTUM, WEIGHT_DECAY = 0.95, 0.1


def _newton_schulz(u, coefficients):
    """The iteration as written, in 32 bits, on a stack of matrices; the Gram on the short side."""
    x = u.mT if u.shape[-2] > u.shape[-1] else u
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    for a, b, c in coefficients:
        gram = torch.bmm(x, x.mT)
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return x.mT if u.shape[-2] > u.shape[-1] else x


def run(state):
    case = state["case"]
    coefficients = COEFFICIENTS[case["coefficients"]]
    if case["op"] == "orthogonalize":
        if own:
            state["plan"].orthogonalize(state["tables"]["grad"], state["tables"]["out"])
        else:
            for g in state["groups"]:
                g["out"].copy_(_newton_schulz(g["grad"].float(), coefficients))
        return [g["out"] for g in state["groups"]]
    if own:
        t = state["tables"]
        state["plan"].muon_step(t["param"], t["grad"], t["velocity"], lr=case["lr"], momentum=MOMENTUM, nesterov=True,
                                weight_decay=WEIGHT_DECAY, scales=state["scales"])
    else:
        for g in state["groups"]:
            grad = g["grad"].float()
            velocity = MOMENTUM * g["velocity"].float() + grad
            update = _newton_schulz(grad + MOMENTUM * velocity, coefficients)
            g["velocity"].copy_(velocity)
            g["param"].copy_(g["param"].float() * (1.0 - case["lr"] * WEIGHT_DECAY) - case["lr"] * g["scale"] * update)
    return [(g["param"], g["velocity"]) for g in state["groups"]]


def work(case):
    to, of, vel = (t.itemsize for t in _types(case))
    elements = sum(count * rows * cols for count, rows, cols in _groups(case))
    each = of + to if case["op"] == "orthogonalize" else of + 2 * to + 2 * vel
    return {"bytes": elements * each, "flops": _flops(case)}


def exact(case, seed):
    """The same from the definition in 64 bits: the polynomial p of the Gram matrix first, its product with X last."""
    state = prepare(case, seed)
    result = []
    for g in state["groups"]:
        grad = g["grad"].double()
        if case["op"] == "muon_step":
            velocity = MOMENTUM * g["velocity"].double() + grad
            u = grad + MOMENTUM * velocity
        else:
            u = grad
        norm = torch.linalg.norm(u.flatten(1), dim=1)[:, None, None] + EPS
        wide = u.shape[1] <= u.shape[2]
        short = u.shape[1] if wide else u.shape[2]
        x = u / norm
        gram = torch.einsum("bij,bkj->bik", x, x) if wide else torch.einsum("bji,bjk->bik", x, x)
        identity = torch.eye(short, dtype=torch.float64, device=u.device)
        p = identity.expand_as(gram)
        for a, b, c in COEFFICIENTS[case["coefficients"]]:
            q = a * identity + gram @ (b * identity + c * gram)
            p, gram = q @ p, q @ gram @ q
        o = p @ x if wide else x @ p
        if case["op"] == "muon_step":
            result.append((g["param"].double() * (1.0 - case["lr"] * WEIGHT_DECAY) - case["lr"] * g["scale"] * o, velocity))
        else:
            result.append(o)
    return result
