"""Operators of a student network that multiplies in 4 bits: what is timed, and their plain forms.

Three families, each beside the layers and losses of `gan_amd.ops`:
  rms_norm             root-mean-square norm with the residual's addition; output in the input's type or in 8 bits (e4m3)
                       with a power-of-two scale per 32 values, the form the product takes
  linear_mx, mx_matmul product of 8- or 4-bit microscaled activations with 4-bit (e2m1) microscaled weights
  distill_topk_mean    loss against a teacher's top logits, fused with its gradient

`own` false: elementary torch operations.  `own` true: the calls a user makes of `gan_amd.ops`.
"""
import math

import torch

own = False

_DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token through a norm that feeds a 4-bit product: launch latency
        dict(name="norm_token", op="norm_serve", rows=1, width=4096, type="bf16", residual=True),
        # a batch of prompts through the same norm
        dict(name="norm_prompt", op="norm_serve", rows=8192, width=4096, type="bf16", residual=True),
        # training on a ragged batch of caption vectors (2400 wide, Text2Image's skip-thought length), half precision
        dict(name="norm_train_ragged", op="norm_train", rows=1023, width=2400, type="f16", residual=False),
        # training of a residual stream
        dict(name="norm_train", op="norm_train", rows=16384, width=2048, type="bf16", residual=True),
        # single token against packed weights
        dict(name="linear_token", op="linear_serve", rows=1, inner=4096, out=4096, type="bf16", fmt="e4m3", given="float"),
        # Text2Image's caption embedding at its batch of 64 (2400 -> 256), fp32 as that model runs
        dict(name="linear_captions", op="linear_serve", rows=64, inner=2400, out=256, type="f32", fmt="e4m3", given="float"),
        # a few sequences decoded together, activations in 4 bits too
        dict(name="linear_few", op="linear_serve", rows=16, inner=8192, out=8192, type="bf16", fmt="e2m1", given="float"),
        # a batch of prompts whose activations come quantised from the norm
        dict(name="linear_prompt", op="linear_serve", rows=4096, inner=8192, out=8192, type="bf16", fmt="e4m3", given="mx"),
        # a training step of one layer: weights quantised, product, three gradients
        dict(name="linear_train", op="linear_train", rows=4096, inner=2048, out=8192, type="bf16", fmt="e4m3"),
        # distillation of a small vocabulary (2500, the command line's default vocab_size) at batch 64
        dict(name="distill_small", op="distill", rows=64, classes=2500, top=16, type="f32", tau=2.0, rest=False, masked=False),
        # distillation of a large vocabulary with the teacher's remaining mass and masked positions
        dict(name="distill_large", op="distill", rows=2048, classes=131072, top=64, type="bf16", tau=1.0, rest=True, masked=True),
        # the operators together: norm -> quantised product -> distillation, forward and backward
        dict(name="student_step", op="student", rows=1024, width=1024, classes=32768, top=32, type="f32", tau=1.5, rest=True,
             masked=True, fmt="e4m3"),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["norm_serve", "norm_train", "linear_serve", "linear_serve", "linear_train", "distill", "distill", "student"])
    typ = rng.choice(["f32", "bf16", "f16"])
    fmt = rng.choice(["e4m3", "e2m1"])
    if op in ("norm_serve", "norm_train"):
        width = spread(33, 16384)
        most = (8192 * 4096 if op == "norm_serve" else 16384 * 2048) * 2 // _BYTES[typ] // width
        return dict(op=op, rows=spread(1, min(16384, most)), width=width, type=typ, residual=rng.random() < 0.5)
    if op == "linear_serve":
        return dict(op=op, rows=spread(1, 4096), inner=spread(33, 8192), out=spread(16, 8192), type=typ, fmt=fmt,
                    given=rng.choice(["float", "mx"]))
    if op == "linear_train":
        return dict(op=op, rows=spread(16, 4096), inner=spread(33, 2048), out=spread(16, 8192), type=typ, fmt=fmt)
    if op == "distill":
        classes = spread(10, 131072)
        return dict(op=op, rows=spread(1, min(8192, 2048 * 131072 * 2 // _BYTES[typ] // classes)), classes=classes,
                    top=spread(1, min(128, classes)), type=typ, tau=rng.choice([1.0, 2.0, 4.0]), rest=rng.random() < 0.5,
                    masked=rng.random() < 0.5)
    classes = spread(256, 32768)
    return dict(op=op, rows=spread(16, 1024), width=spread(64, 1024), classes=classes, top=spread(1, min(128, classes)), type="f32",
                tau=rng.choice([1.0, 2.0]), rest=rng.random() < 0.5, masked=rng.random() < 0.5, fmt="e4m3")


def work(case):
    b, op = _BYTES[case["type"]], case["op"]
    r = case["rows"]
    if op == "norm_serve":
        n = r * case["width"]
        return {"bytes": n * ((3 if case["residual"] else 1) * b + 1 + 1 / 32) + 4 * case["width"], "flops": 8 * n}
    if op == "norm_train":
        n = r * case["width"]
        return {"bytes": n * (7 if case["residual"] else 4) * b + 8 * case["width"], "flops": 16 * n}
    if op == "linear_serve":
        k, n = case["inner"], case["out"]
        code = (1 if case["fmt"] == "e4m3" else 0.5) + 1 / 32
        return {"bytes": r * k * (b if case["given"] == "float" else code) + k * n * (0.5 + 1 / 32) + 4 * n + r * n * b,
                "flops": 2 * r * k * n}
    if op == "linear_train":
        k, n = case["inner"], case["out"]
        return {"bytes": 2 * r * k * b + 8 * k * n + 8 * n + 2 * r * n * b, "flops": 6 * r * k * n}
    lists = r * case["top"] * (b + 4) + (4 * r if case["rest"] else 0) + (4 * r if case["masked"] else 0)
    if op == "distill":
        return {"bytes": 2 * r * case["classes"] * b + lists + 4, "flops": 10 * r * case["classes"]}
    k, n = case["width"], case["classes"]
    return {"bytes": 4 * r * k * b + 8 * k * n + 8 * n + 8 * k + lists + 4, "flops": 6 * r * k * n}


# ------------------------------------------------------------------------------------------------ microscaled values
def _blocks(x):
    """[..., K] as [..., K/32, 32], the last block filled with zeros."""
    k = x.shape[-1]
    return torch.nn.functional.pad(x, (0, -k % 32)).reshape(x.shape[:-1] + (-1, 32))


def _quantise(x, fmt):
    """Element values and scales of fp32 `x` in blocks of 32 along its last axis: the scale is the smallest power of two (from
    2^-126 on) under which the block's largest magnitude is no larger than the format's (448 e4m3, 6 e2m1)."""
    v = _blocks(x)
    mant, ex = torch.frexp(v.abs().amax(-1, keepdim=True))
    e = ex - 9 + (mant > 0.875) if fmt == "e4m3" else ex - 3 + (mant > 0.75)
    e = e.clamp(-126, 127)
    v = torch.ldexp(v, -e)
    if fmt == "e4m3":
        v = v.to(torch.float8_e4m3fn).float()
    else:
        a = v.abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        v = torch.copysign(torch.round(a / step) * step, v)
    return v, torch.ldexp(torch.ones_like(x[..., :1, None]).expand(e.shape), e)


def _values(v, scale, width):
    return (v * scale).flatten(-2)[..., :width]


def _mx(x, fmt):
    """What the microscaled form of fp32 `x` stands for."""
    v, scale = _quantise(x, fmt)
    return _values(v, scale, x.shape[-1])


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nibbles(v):
    """4-bit codes of e2m1 values, two to a byte, the first in the low half."""
    table = torch.tensor(_E2M1, device=v.device)
    code = torch.bucketize(v.abs(), table) | (torch.signbit(v).long() << 3)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8)


def _pad_to(x, axis, n):
    out = torch.zeros(x.shape[:axis] + (n,) + x.shape[axis + 1:], dtype=x.dtype, device=x.device)
    out.narrow(axis, 0, x.shape[axis]).copy_(x)
    return out


def _scale_bytes(scale):
    return (torch.frexp(scale)[1] - 1 + 127).to(torch.uint8)


# ------------------------------------------------------------------------------------------------ inputs
def _lists(case, g, dev, typ):
    """A teacher's top classes of every row: one class in each of `top` equal ranges, logits in falling order, some left out."""
    r, c, k = case["rows"], case["classes"], case["top"]
    width = c // k
    index = torch.arange(k, device=dev) * width + torch.randint(0, width, (r, k), generator=g, device=dev)
    index = torch.gather(index, 1, torch.rand(r, k, generator=g, device=dev).argsort(1))
    teacher = (torch.randn(r, k, generator=g, device=dev) * 2).sort(1, descending=True)[0]
    s = dict(index=index.to(torch.int32), teacher=teacher.to(typ), lse=None, weight=None)
    if case["masked"]:      # lists of different lengths, and rows that do not count
        length = torch.randint(max(1, k // 2), k + 1, (r, 1), generator=g, device=dev)
        s["index"] = torch.where(torch.arange(k, device=dev) < length, s["index"], torch.full_like(s["index"], -1))
        s["weight"] = (torch.rand(r, generator=g, device=dev) < 0.9).float()
        s["weight"][:1] = 1.0
    if case["rest"]:        # the teacher's whole normaliser: its list holds 60 to 95 % of the mass
        t = torch.where(s["index"] >= 0, s["teacher"].float() / case["tau"], -math.inf)
        held = 0.6 + 0.35 * torch.rand(r, generator=g, device=dev)
        top = t.amax(1)
        s["lse"] = top + torch.exp(t - top[:, None]).sum(1).log() - held.log()
    return s


def prepare(case, seed):
    dev = _DEVICE
    g = torch.Generator(device=dev).manual_seed(int(seed))
    typ, r, op = _TYPES[case["type"]], case["rows"], case["op"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": case}
    if op in ("norm_serve", "norm_train", "student"):
        w = case["width"]
        s["x"] = normal(r, w).to(typ)
        if op == "student" or case["residual"]:
            s["r"] = (2 * normal(r, w)).to(typ)
        s["gamma"] = 1 + 0.1 * normal(w)
    if op == "norm_train":
        s["dy"] = normal(r, case["width"]).to(typ)
        s["dh"] = normal(r, case["width"]).to(typ) if case["residual"] else None
    if op in ("linear_serve", "linear_train"):
        k, n = case["inner"], case["out"]
        x = normal(r, k).to(typ)
        matrix = normal(k, n) / math.sqrt(k)
        s["bias"] = 0.1 * normal(n)
        if op == "linear_train":
            s.update(x=x, matrix=matrix, dy=normal(r, n).to(typ))
        else:
            # weights as a serving program keeps them: packed once, [blocks][out][16 bytes] and [blocks / 4][out][4] scale bytes
            # with the blocks filled up to a multiple of 4; beside them the values for a program that multiplies in 32 bits
            v, scale = _quantise(matrix.t().contiguous(), "e2m1")
            s["matrix"] = _values(v, scale, k).t().contiguous()
            nb = -(-v.shape[1] // 4) * 4
            codes = _pad_to(_nibbles(v), 1, nb)
            byte = _pad_to(_scale_bytes(scale[..., 0]), 1, nb)
            s["codes"] = codes.transpose(0, 1).contiguous()
            s["scales"] = byte.reshape(n, nb // 4, 4).transpose(0, 1).contiguous()
            if case["given"] == "float":
                s["x"] = x
            else:           # activations as a norm leaves them: rows filled up with zeros to a multiple of 128 values
                v, scale = _quantise(x.float(), case["fmt"])
                flat = v.flatten(1).to(torch.float8_e4m3fn).view(torch.uint8) if case["fmt"] == "e4m3" else _nibbles(v).flatten(1)
                s["x_codes"] = _pad_to(flat, 1, nb * (32 if case["fmt"] == "e4m3" else 16))
                s["x_scales"] = _pad_to(_scale_bytes(scale[..., 0]), 1, nb)
    if op == "distill":
        s["logits"] = (2 * normal(r, case["classes"])).to(typ)
    if op == "student":
        s["matrix"] = 2 * normal(case["width"], case["classes"]) / math.sqrt(case["width"])
        s["bias"] = 0.1 * normal(case["classes"])
    if op in ("distill", "student"):
        s.update(_lists(case, g, dev, typ))
    if own:
        _handles(s)
    return s


def _handles(s):
    """What a program of this framework keeps besides its inputs: variables in their store, and the object that names packed
    weights.  Nothing is computed here."""
    from gan_amd import ops
    from gan_amd import variables as V
    case, op = s["case"], s["case"]["op"]
    if op == "linear_serve":
        s["packed"] = ops.MxMatrix(s["codes"], s["scales"], case["inner"], case["out"])
        if case["given"] == "mx":
            s["mx"] = ops.MxTensor(s["x_codes"], s["x_scales"], case["inner"], case["fmt"], _TYPES[case["type"]])
        return
    if op == "distill":
        return
    store = V.VariableStore(device=_DEVICE)
    with V.use_store(store):
        if "gamma" in s:
            with store.variable_scope("rms_norm"):
                store.get_variable("gamma", [case["width"]], V.constant_initializer(1.0)).data.copy_(s["gamma"])
        if "matrix" in s:
            k, n = s["matrix"].shape
            with store.variable_scope("Linear"):
                store.get_variable("Matrix", [k, n], V.constant_initializer(0.0)).data.copy_(s["matrix"])
                store.get_variable("bias", [n], V.constant_initializer(0.0)).data.copy_(s["bias"])
    s["store"], s["group"] = store, store.pack("layers", store.trainable_variables())


# ------------------------------------------------------------------------------------------------ plain forms
def _norm64(h, gamma):
    """y in 64 bits: a value next to a border of the 8-bit grid has to fall on its own side."""
    h = h.double()
    return (h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * gamma.double()).float()


def _stream(s, typ):
    """The residual stream as it is stored, in the tensors' type."""
    return (s["x"].float() + s["r"].float()).to(typ) if "r" in s else s["x"]


def _norm_backward(h, gamma, dy, dh):
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    n = h * rstd
    g = dy * gamma
    dx = rstd * (g - n * (g * n).mean(1, keepdim=True))
    return dx if dh is None else dx + dh, (dy * n).sum(0)


def _distill(logits, s):
    """Loss and its gradient with respect to fp32 `logits`."""
    case = s["case"]
    tau, classes = case["tau"], logits.shape[1]
    index, t = s["index"].long(), s["teacher"].float() / tau
    valid = (index >= 0) & (index < classes)
    w = torch.ones(logits.shape[0], device=logits.device) if s["weight"] is None else s["weight"]
    w = torch.where(valid.any(1), w, 0.0)
    total = w.numel() if s["weight"] is None else s["weight"].sum()
    t = torch.where(valid, t, -math.inf)
    if s["lse"] is None:
        top = t.amax(1, keepdim=True)
        logp = t - top - torch.exp(t - top).sum(1, keepdim=True).log()
    else:
        logp = t - s["lse"][:, None]
    p = torch.exp(logp)
    z = logits / tau
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    norm = e.sum(1, keepdim=True)
    logq = torch.gather(z, 1, index.clamp(0, classes - 1)) - top - norm.log()
    loss = torch.where(valid, p * (logp - logq), 0.0).sum(1)
    place = torch.where(valid, index, classes)
    target = torch.zeros(z.shape[0], classes + 1, device=z.device).scatter_add_(1, place, torch.where(valid, p, 0.0))[:, :classes]
    mass = p.sum(1, keepdim=True)
    if s["lse"] is None:
        grad = e / norm - target
    else:
        rest = (1 - mass).clamp(min=0)
        listed_ = torch.zeros(z.shape[0], classes + 1, dtype=torch.bool, device=z.device).scatter_(1, place, True)[:, :classes]
        zu = torch.where(listed_, -math.inf, z)
        topu = zu.amax(1, keepdim=True)
        eu = torch.exp(zu - topu)
        normu = eu.sum(1, keepdim=True)
        there = (rest > 0) & (topu > -math.inf)
        logqr = topu + normu.log() - top - norm.log()
        loss = loss + torch.where(there, rest * (rest.log() - logqr), 0.0)[:, 0]
        grad = (mass + rest) * (e / norm) - target - torch.where(there, rest * (eu / normu), 0.0)
    scale = w / total
    return (tau * tau * (loss * scale).sum()).reshape(1), torch.where(w[:, None] != 0, grad * (tau * scale[:, None]), 0.0)


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    typ = _TYPES[case["type"]]
    if op == "norm_serve":
        h = _stream(s, typ)
        v, scale = _quantise(_norm64(h, s["gamma"]), "e4m3")
        out = {"codes": v.flatten(1)[:, :case["width"]].to(torch.float8_e4m3fn), "scales": scale[..., 0].to(torch.float8_e8m0fnu)}
        return dict(out, h=h) if case["residual"] else out
    if op == "norm_train":
        h = _stream(s, typ)
        h32 = h.float()
        y = h32 * torch.rsqrt((h32 * h32).mean(1, keepdim=True) + EPS) * s["gamma"]
        dx, dgamma = _norm_backward(h32, s["gamma"], s["dy"].float(), None if s["dh"] is None else s["dh"].float())
        out = {"y": y.to(typ), "dx": dx.to(typ), "dgamma": dgamma}
        return dict(out, h=h) if case["residual"] else out
    if op == "linear_serve":
        if case["given"] == "float":
            a = _mx(s["x"].float(), case["fmt"])
        else:
            if case["fmt"] == "e4m3":
                v = s["x_codes"].view(torch.float8_e4m3fn).float()
            else:
                both = torch.stack([s["x_codes"] & 15, s["x_codes"] >> 4], -1).flatten(1).long()
                table = torch.tensor(_E2M1 + tuple(-t for t in _E2M1), device=both.device)
                v = table[both]
            a = (v.unflatten(1, (-1, 32)) * s["x_scales"].view(torch.float8_e8m0fnu).float()[..., None]).flatten(1)[:, :case["inner"]]
        return (torch.matmul(a, s["matrix"]) + s["bias"]).to(typ)
    if op == "linear_train":
        a, w, dy = _mx(s["x"].float(), case["fmt"]), _mx(s["matrix"].t().contiguous(), "e2m1").t(), s["dy"].float()
        return {"y": (torch.matmul(a, w) + s["bias"]).to(typ), "dx": torch.matmul(dy, w.t()).to(typ),
                "dmatrix": torch.matmul(a.t(), dy), "dbias": dy.sum(0)}
    if op == "distill":
        loss, grad = _distill(s["logits"].float(), s)
        return {"loss": loss, "dlogits": grad.to(typ)}
    h = _stream(s, typ)
    a, w = _mx(_norm64(h, s["gamma"]), case["fmt"]), _mx(s["matrix"].t().contiguous(), "e2m1").t()
    loss, dlogits = _distill(torch.matmul(a, w) + s["bias"], s)
    dx, dgamma = _norm_backward(h.float(), s["gamma"], torch.matmul(dlogits, w.t()), None)
    return {"loss": loss, "h": h, "dx": dx, "dgamma": dgamma, "dmatrix": torch.matmul(a.t(), dlogits), "dbias": dlogits.sum(0)}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from gan_amd import ops
    from gan_amd import variables as V
    case, op = s["case"], s["case"]["op"]
    if op == "norm_serve":
        with V.use_store(s["store"]), torch.no_grad():
            out = ops.rms_norm(s["x"], residual=s.get("r"), epsilon=EPS, mx=True)
        q, h = out if case["residual"] else (out, None)
        out = {"codes": q.codes[:, :case["width"]], "scales": q.scales[:, :-(-case["width"] // 32)]}
        return dict(out, h=h) if case["residual"] else out
    if op == "linear_serve":
        return ops.mx_matmul(s["x"] if case["given"] == "float" else s["mx"], s["packed"], s["bias"], fmt=case["fmt"])
    if op == "distill":
        logits = s["logits"].detach().requires_grad_(True)
        loss = ops.distill_topk_mean(logits, s["teacher"], s["index"], temperature=case["tau"], row_weight=s["weight"],
                                     teacher_lse=s["lse"])
        ops.backward(loss)
        return {"loss": loss.detach(), "dlogits": logits.grad}
    store, group = s["store"], s["group"]
    with V.use_store(store):
        group.begin_update()
        x = s["x"].detach().requires_grad_(True)
        if op == "norm_train":
            y = ops.rms_norm(x, residual=s.get("r"), epsilon=EPS)
            if case["residual"]:
                y, h = y
                torch.autograd.backward((y, h), (s["dy"], s["dh"]))
                out = {"y": y.detach(), "h": h.detach()}
            else:
                torch.autograd.backward((y,), (s["dy"],))
                out = {"y": y.detach()}
            out["dgamma"] = store.vars["rms_norm/gamma"].grad
        elif op == "linear_train":
            y = ops.linear_mx(x, case["out"], fmt=case["fmt"])
            torch.autograd.backward((y,), (s["dy"],))
            out = {"y": y.detach(), "dmatrix": store.vars["Linear/Matrix"].grad, "dbias": store.vars["Linear/bias"].grad}
        else:
            q, h = ops.rms_norm(x, residual=s["r"], epsilon=EPS, mx=True)
            logits = ops.linear_mx(q, case["classes"])
            loss = ops.distill_topk_mean(logits, s["teacher"], s["index"], temperature=case["tau"], row_weight=s["weight"],
                                         teacher_lse=s["lse"])
            ops.backward(loss)
            out = {"loss": loss.detach(), "h": h.detach(), "dgamma": store.vars["rms_norm/gamma"].grad,
                   "dmatrix": store.vars["Linear/Matrix"].grad, "dbias": store.vars["Linear/bias"].grad}
        group.end_update()
        out["dx"] = x.grad
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def _grid(fmt):
    """The format's values of positive sign, by code."""
    if fmt == "e2m1":
        return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119]


def _snap(x, fmt):
    """Element values [.., blocks, 32] and scales [.., blocks] of 64-bit x: nearest value of the grid, ties to the even code."""
    grid = torch.tensor(_grid(fmt), dtype=torch.float64, device=x.device)
    b = torch.zeros(x.shape[:-1] + (-(-x.shape[-1] // 32) * 32,), dtype=torch.float64, device=x.device)
    b[..., :x.shape[-1]] = x
    b = b.unflatten(-1, (-1, 32))
    e = torch.ceil(torch.log2(b.abs().max(-1)[0] / grid[-1])).clamp(-126, 127)
    scale = torch.exp2(e)
    b = b / scale[..., None]
    middle = (grid[1:] + grid[:-1]) / 2
    a = b.abs()
    below = torch.bucketize(a, middle, out_int32=True)
    above = torch.bucketize(a, middle, right=True, out_int32=True)
    return torch.sign(b) * grid[torch.where(below % 2 == 0, below, above).long()], scale


def _snapped(x, fmt):
    v, scale = _snap(x, fmt)
    return (v * scale[..., None]).flatten(-2)[..., :x.shape[-1]]


def _stored(s):
    if "r" not in s:
        return s["x"].double()
    total = s["x"].double() + s["r"].double()
    return total if s["x"].dtype == torch.float64 else total.to(s["x"].dtype).double()


def _normed(h, gamma):
    root = torch.sqrt(torch.sum(h ** 2, 1) / h.shape[1] + EPS)
    return h / root[:, None], root


def _normed_gradients(h, gamma, dy, dh):
    n, root = _normed(h, gamma)
    g = dy * gamma
    dx = (g - n * (torch.sum(g * n, 1) / h.shape[1])[:, None]) / root[:, None]
    return (dx if dh is None else dx + dh), torch.einsum("rc,rc->c", dy, n)


def _distilled(logits, s):
    """From log q = z - log sum exp z over all classes; the gradient as the sum of its parts."""
    case, rows = s["case"], logits.shape[0]
    tau, classes = case["tau"], logits.shape[1]
    logq = logits / tau
    logq = logq - torch.logsumexp(logq, 1, keepdim=True)
    row, col = torch.nonzero((s["index"] >= 0) & (s["index"] < classes), as_tuple=True)
    t = torch.full(s["index"].shape, -math.inf, dtype=torch.float64, device=logits.device)
    t[row, col] = s["teacher"].double()[row, col] / tau
    norm = torch.logsumexp(t, 1) if s["lse"] is None else s["lse"].double()
    at = s["index"].long()[row, col]
    logp = t[row, col] - norm[row]
    p = torch.exp(logp)
    loss = torch.zeros(rows, dtype=torch.float64, device=logits.device).index_add_(0, row, p * (logp - logq[row, at]))
    mass = torch.zeros(rows, dtype=torch.float64, device=logits.device).index_add_(0, row, p)
    rest = torch.zeros_like(mass) if s["lse"] is None else torch.clamp(1 - mass, min=0)
    q = torch.exp(logq)
    grad = q * (mass + rest)[:, None]
    if s["lse"] is not None:
        logq[row, at] = -math.inf
        outside = torch.logsumexp(logq, 1)
        there = (rest > 0) & torch.isfinite(outside)
        loss += torch.where(there, torch.xlogy(rest, rest) - rest * torch.where(there, outside, 0.0), 0.0)
        logq -= torch.where(there, outside, 0.0)[:, None]
        grad -= torch.where(there, rest, 0.0)[:, None] * logq.exp_()
    grad.index_put_((row, at), -p, accumulate=True)
    w = torch.ones(rows, dtype=torch.float64, device=logits.device) if s["weight"] is None else s["weight"].double()
    share = w / w.sum()
    share = torch.where((s["index"] >= 0).any(1), share, 0.0)
    return (tau ** 2 * torch.dot(share, loss)).reshape(1), grad * (tau * share)[:, None]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    gamma = s["gamma"].double() if "gamma" in s else None
    if op == "norm_serve":
        h = _stored(s)
        v, scale = _snap(_normed(h, gamma)[0] * gamma, "e4m3")
        out = {"codes": v.flatten(1)[:, :case["width"]], "scales": scale}
        return dict(out, h=h) if case["residual"] else out
    if op == "norm_train":
        h = _stored(s)
        dx, dgamma = _normed_gradients(h, gamma, s["dy"].double(), None if s["dh"] is None else s["dh"].double())
        out = {"y": _normed(h, gamma)[0] * gamma, "dx": dx, "dgamma": dgamma}
        return dict(out, h=h) if case["residual"] else out
    if op == "linear_serve":
        if case["given"] == "float":
            a = _snapped(s["x"].double(), case["fmt"])
        else:
            grid = torch.tensor(_grid(case["fmt"]), dtype=torch.float64, device=s["x_codes"].device)
            c = s["x_codes"].long()
            if case["fmt"] == "e2m1":
                c = torch.stack((c % 16, c // 16), 2).reshape(c.shape[0], -1)
            half = 8 if case["fmt"] == "e2m1" else 128
            v = torch.where(c >= half, -1.0, 1.0) * grid[(c % half).clamp(max=grid.numel() - 1)]
            a = v * torch.exp2(s["x_scales"].double() - 127).repeat_interleave(32, 1)
            a = a[:, :case["inner"]]
        return a @ s["matrix"].double() + s["bias"].double()
    if op == "linear_train":
        a, w, dy = _snapped(s["x"].double(), case["fmt"]), _snapped(s["matrix"].double().t(), "e2m1"), s["dy"].double()
        return {"y": a @ w.t() + s["bias"].double(), "dx": dy @ w, "dmatrix": a.t() @ dy, "dbias": dy.sum(0)}
    if op == "distill":
        loss, grad = _distilled(s["logits"].double(), s)
        return {"loss": loss, "dlogits": grad}
    h = _stored(s)
    a, w = _snapped(_normed(h, gamma)[0] * gamma, case["fmt"]), _snapped(s["matrix"].double().t(), "e2m1")
    loss, dlogits = _distilled(a @ w.t() + s["bias"].double(), s)
    dx, dgamma = _normed_gradients(h, gamma, dlogits @ w, None)
    return {"loss": loss, "h": h, "dx": dx, "dgamma": dgamma, "dmatrix": a.t() @ dlogits, "dbias": dlogits.sum(0)}
