"""The operators at the head of a network, as measurable cases: layer normalisation, the logits that a teacher keeps, distillation from
them, and categories drawn from logits.

Buffers are node-major and frame-minor, as everywhere in this framework: [nodes, pitch] rows of fp32 frames or packed bits, nodes of the
classifier's operators being (channel, pixel).  Each operator has its plain form (elementary torch operations in 32 bits, the draw in 64)
beside the framework's call.
"""
import math

import torch

own = False

EPS = 1.0e-5


# ---- what is measured ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one frame of a served network: latency
        {"name": "layer norm, one frame", "op": "ln_forward", "nodes": 1024, "frames": 1, "bits": False},
        # the hidden layer of the classifier's training step, packed activations
        {"name": "layer norm, packed bits", "op": "ln_forward", "nodes": 6144, "frames": 1024, "bits": True},
        # the headline layer's activations
        {"name": "layer norm, large", "op": "ln_forward", "nodes": 4096, "frames": 8192, "bits": False},
        # a training step at an odd batch
        {"name": "layer norm backward", "op": "ln_backward", "nodes": 1024, "frames": 1000, "bits": False},
        {"name": "layer norm backward, large", "op": "ln_backward", "nodes": 4096, "frames": 8192, "bits": False},
        # a teacher's pass over images: few classes at each of 32 x 32 pixels
        {"name": "top logits of pixels", "op": "top", "channels": 21, "pixels": 1024, "frames": 65, "top": 5, "rounded": False},
        # a teacher with many classes, whose logits were computed in 16 bits: equal values are frequent
        {"name": "top logits, many channels", "op": "top", "channels": 32768, "pixels": 1, "frames": 1024, "top": 64, "rounded": True},
        # the smallest training step: ten classes, 64 frames
        {"name": "distillation, ten classes", "op": "distill", "channels": 10, "pixels": 1, "frames": 64, "top": 4, "temperature": 4.0},
        {"name": "distillation, odd sizes", "op": "distill", "channels": 1001, "pixels": 1, "frames": 777, "top": 17, "temperature": 2.0},
        {"name": "distillation, many channels", "op": "distill", "channels": 32768, "pixels": 1, "frames": 2048, "top": 64, "temperature": 1.5},
        # one request of a server
        {"name": "sampling, one frame", "op": "sample", "channels": 32768, "pixels": 1, "frames": 1, "top": 50, "temperature": 0.8, "top_p": 0.95, "min_p": 0.0},
        # a batch of requests
        {"name": "sampling, a batch", "op": "sample", "channels": 10007, "pixels": 1, "frames": 256, "top": 40, "temperature": 1.0, "top_p": 0.9, "min_p": 0.05},
    ]


def _size(rng, lo, hi):
    """spread over the logarithm of the range"""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["ln_forward", "ln_backward", "top", "distill", "sample"])
    if op in ("ln_forward", "ln_backward"):
        nodes = _size(rng, 2, 16384)
        return {"op": op, "nodes": nodes, "frames": _size(rng, 1, min(16384, (1 << 25) // nodes)), "bits": rng.random() < 0.25}
    channels = _size(rng, 2, 32768)
    pixels = _size(rng, 2, 1024) if channels <= 256 and rng.random() < 0.5 else 1
    frames = _size(rng, 1, min(8192, (1 << 25) // (channels * pixels)))
    case = {"op": op, "channels": channels, "pixels": pixels, "frames": frames, "top": min(channels, _size(rng, 1, 256))}
    if op == "top":
        case["rounded"] = rng.random() < 0.5
    else:
        case["temperature"] = round(rng.uniform(0.5, 4.0), 3)
    if op == "sample":
        case["top_p"] = 1.0 if rng.random() < 0.3 else round(rng.uniform(0.3, 0.99), 3)
        case["min_p"] = 0.0 if rng.random() < 0.5 else round(rng.uniform(0.01, 0.3), 3)
    return case


def _pitch(frames):
    """floats from row to row, as the framework's buffers have them: whole 256 bytes, not a multiple of 2 KiB"""
    p = (frames + 63) // 64 * 64
    return p + 128 if p % 512 == 0 else p


def _words(frames):
    p = (frames + 2047) // 2048 * 64
    return p + 96 if p % 512 == 0 else p


def work(case):
    if case["op"] in ("ln_forward", "ln_backward"):
        n, f = case["nodes"], case["frames"]
        x = n * f / 8 if case["bits"] else 4 * n * f
        if case["op"] == "ln_forward":
            return {"bytes": x + 4 * n * f + 8 * n + 8 * f, "flops": 8 * n * f}
        return {"bytes": x + 8 * n * f + 12 * n + 8 * f, "flops": 14 * n * f}
    columns, c, k = case["pixels"] * case["frames"], case["channels"], case["top"]
    if case["op"] == "top":
        return {"bytes": columns * (4 * c + 8 * k), "flops": columns * c}
    if case["op"] == "distill":
        return {"bytes": columns * (8 * c + 8 * k + 8), "flops": columns * (8 * c + 16 * k)}
    return {"bytes": columns * (4 * c + 12), "flops": columns * (c + 16 * k)}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------
def _rows(gen, nodes, frames, scale=1.0):
    """[nodes, pitch] frames; what lies behind a row's last frame is nobody's"""
    return torch.randn((nodes, _pitch(frames)), generator=gen, device="cuda").mul_(scale)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    f = case["frames"]
    state = dict(case)
    if case["op"] in ("ln_forward", "ln_backward"):
        n = case["nodes"]
        if case["bits"]:
            state["x"] = torch.randint(-(1 << 31), 1 << 31, (n, _words(f)), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
        else:
            state["x"] = _rows(gen, n, f).add_(0.5)
        state["gamma"] = 1.0 + 0.1 * torch.randn(n, generator=gen, device="cuda")
        state["beta"] = 0.1 * torch.randn(n, generator=gen, device="cuda")
        if case["op"] == "ln_backward":
            state["dy"] = _rows(gen, n, f)
            v = _values(state).double()
            state["mean"] = v.mean(0).float()
            state["rstd"] = (1.0 / torch.sqrt(v.var(0, unbiased=False) + EPS)).float()
        return state
    c, p, k = case["channels"], case["pixels"], case["top"]
    y = _rows(gen, c * p, f, 3.0)
    if case.get("rounded"):
        y = y.to(torch.bfloat16).float()
    state["y"] = y
    if case["op"] == "distill":
        # a teacher that mostly agrees, its record shorter in every fifth frame; every eighth frame is padding of the batch
        teacher = y.view(c, p, -1) + torch.randn((c, p, y.shape[1]), generator=gen, device="cuda")
        z, index = torch.topk(teacher, k, dim=0)
        index = index.to(torch.int32)
        index[k // 2 + 1:, :, ::5] = -1
        state["index"], state["logit"] = index.reshape(k * p, -1).contiguous(), z.reshape(k * p, -1).contiguous()
        weight = torch.rand((p, y.shape[1]), generator=gen, device="cuda") + 0.5
        weight[:, 7::8] = 0.0
        state["weight"], state["weight_sum"] = weight, float(weight[:, :f].double().sum())
    if case["op"] == "sample":
        state["u"] = torch.rand((p, y.shape[1]), generator=gen, device="cuda")
    return state


def _values(s):
    """the input of a normalisation as fp32 [nodes, frames]"""
    x, f = s["x"], s["frames"]
    if not s["bits"]:
        return x[:, :f]
    bit = torch.arange(32, device=x.device, dtype=torch.int32)
    return ((x[:, :(f + 31) // 32, None] >> bit) & 1).reshape(x.shape[0], -1)[:, :f].float()


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(state):
    return {"ln_forward": _ln_forward, "ln_backward": _ln_backward, "top": _top, "distill": _distill, "sample": _sample}[state["op"]](state)


def _ln_forward(s):
    f = s["frames"]
    if own:
        from binarybrain_amd import ops
        if s["bits"]:
            y, mean, rstd = ops.bit_layer_normalization_forward(s["x"], s["gamma"], s["beta"], f, _pitch(f), eps=EPS)
        else:
            y, mean, rstd = ops.layer_normalization_forward(s["x"], s["gamma"], s["beta"], f, eps=EPS)
        return y[:, :f], mean, rstd
    v = _values(s)
    mean = v.mean(0)
    d = v - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(0) + EPS)
    return d * rstd * s["gamma"][:, None] + s["beta"][:, None], mean, rstd


def _ln_backward(s):
    f = s["frames"]
    if own:
        from binarybrain_amd import ops
        call = ops.bit_layer_normalization_backward if s["bits"] else ops.layer_normalization_backward
        dx, dgamma, dbeta = call(s["x"], s["dy"], s["gamma"], s["mean"], s["rstd"], f)
        return dx[:, :f], dgamma, dbeta
    dy = s["dy"][:, :f]
    xh = (_values(s) - s["mean"]) * s["rstd"]
    g = dy * s["gamma"][:, None]
    dx = s["rstd"] * (g - g.mean(0) - xh * (g * xh).mean(0))
    return dx, (dy * xh).sum(1), dy.sum(1)


def _columns(t, rows, s):
    """[rows * pixels, pitch] as [rows, pixels, frames]"""
    return t.view(rows, s["pixels"], t.shape[1])[:, :, :s["frames"]]


def _largest(s):
    """the largest logits of each column, descending, of equal ones the lowest channel first: (channels, values) [top, pixels, frames]"""
    value, channel = torch.sort(_columns(s["y"], s["channels"], s), dim=0, descending=True, stable=True)
    return channel[:s["top"]], value[:s["top"]]


def _top(s):
    f, k = s["frames"], s["top"]
    if own:
        from binarybrain_amd import ops
        index, logit = ops.top_logits(s["y"], k, s["channels"], s["pixels"], f)
        return index[:, :f], logit[:, :f]
    channel, value = _largest(s)
    return channel.to(torch.int32).reshape(k * s["pixels"], f), value.reshape(k * s["pixels"], f)


def _distill(s):
    f, c, p, k, t = s["frames"], s["channels"], s["pixels"], s["top"], s["temperature"]
    if own:
        from binarybrain_amd import ops
        dy, loss = ops.loss_distillation(s["y"], s["index"], s["logit"], c, p, f, temperature=t, weight=s["weight"], weight_sum=s["weight_sum"])
        return dy[:, :f], loss[:, :f]
    y, index, z = _columns(s["y"], c, s) / t, _columns(s["index"], k, s), _columns(s["logit"], k, s) / t
    w = s["weight"][:, :f]
    shifted = y - y.amax(0)
    e = torch.exp(shifted)
    total = e.sum(0)
    listed_ = (index >= 0) & (index < c)
    at = torch.where(listed_, index, 0).long()
    z = torch.where(listed_, z, -math.inf)
    top = z.amax(0)
    empty = top == -math.inf
    ez = torch.where(listed_, torch.exp(z - torch.where(empty, 0.0, top)), 0.0)
    q = ez / torch.where(empty, 1.0, ez.sum(0))
    log_ratio = torch.log(torch.where(q > 0, q, 1.0)) - (shifted.gather(0, at) - torch.log(total))
    none = empty | (w == 0)
    loss = torch.where(none, 0.0, w * (t * t) * torch.where(q > 0, q * log_ratio, 0.0).sum(0))
    dy = torch.where(none, 0.0, (e / total).scatter_add(0, at, -q) * (w * (t / s["weight_sum"])))
    return dy.reshape(c * p, f), loss


def _sample(s):
    f, k = s["frames"], s["top"]
    if own:
        from binarybrain_amd import ops
        category, share = ops.categorical_sampling(s["y"], s["u"], s["channels"], s["pixels"], f, temperature=s["temperature"], top_size=k,
                                                   top_p=s["top_p"], min_p=s["min_p"])
        return category[:, :f], share[:, :f]
    channel, value = _largest(s)
    value, u = value.double(), s["u"][:, :f].double()
    # (scalars as the framework's calls take them: rounded to 32 bits)
    t, top_p, min_p = (float(torch.tensor(s[name], dtype=torch.float32)) for name in ("temperature", "top_p", "min_p"))
    e = torch.exp((value - value[0]) / t)
    up_to = e.cumsum(0)
    kept = (e > 0) & (e >= min_p)
    if top_p < 1.0:
        kept &= torch.cat([torch.ones_like(kept[:1]), up_to[:-1] < top_p * up_to[-1]])
    count = kept.sum(0)                                          # a prefix: every rule keeps the first so many
    total = up_to.gather(0, count[None] - 1)[0]
    at = torch.minimum(((up_to <= u * total) & kept).sum(0), count - 1)[None]
    return channel.gather(0, at)[0].to(torch.int32), (e.gather(0, at)[0] / total).float()


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op, f = case["op"], case["frames"]
    if op in ("ln_forward", "ln_backward"):
        n = case["nodes"]
        x = _values(s).to(torch.float64)
        gamma, beta = s["gamma"].double().unsqueeze(1), s["beta"].double().unsqueeze(1)
        if op == "ln_forward":
            mean = x.sum(0) / n
            rstd = ((x - mean).square().sum(0) / n + EPS).rsqrt()
            return (x - mean).mul(rstd).mul(gamma).add(beta), mean, rstd
        mean, rstd, dy = s["mean"].double(), s["rstd"].double(), s["dy"][:, :f].double()
        xh = (x - mean) * rstd
        a = (dy * gamma).sum(0) / n
        b = (dy * gamma * xh).sum(0) / n
        return rstd * (dy * gamma) - rstd * a - rstd * xh * b, (dy * xh).sum(1), dy.sum(1)
    c, p, k = case["channels"], case["pixels"], case["top"]
    y = s["y"].double().reshape(c, p, -1)[:, :, :f]
    if op == "top":
        return None, torch.topk(y, k, dim=0, sorted=True).values.reshape(k * p, f)
    t = case["temperature"]
    if op == "distill":
        index, z, w = s["index"].reshape(k, p, -1)[:, :, :f].long(), s["logit"].double().reshape(k, p, -1)[:, :, :f], s["weight"][:, :f].double()
        log_p = torch.log_softmax(y / t, 0)
        log_q = torch.log_softmax(torch.where(index >= 0, z / t, -math.inf), 0)
        q = log_q.exp()
        there = index.clamp_min(0)
        loss = (q * torch.where(q > 0, log_q - log_p.gather(0, there), 0.0)).sum(0) * w * t * t
        dense = torch.zeros_like(y).scatter_add_(0, there, q)
        return ((log_p.exp() - dense) * (w * t / s["weight_sum"])).reshape(c * p, f), loss
    # the share of the category that the definition draws: prefix by prefix of the sorted probabilities
    t32, top_p, min_p = (float(torch.tensor(case[name], dtype=torch.float32)) for name in ("temperature", "top_p", "min_p"))
    best = torch.topk(y, k, dim=0, sorted=True).values
    prob = torch.softmax(best / t32, 0)
    gone = torch.cumsum(prob, 0) - prob                          # the mass before each
    ok = (prob >= min_p * prob[0]) & ((gone < top_p) if top_p < 1.0 else torch.ones_like(prob, dtype=torch.bool))
    ok[0] = True
    prob = torch.where(ok, prob, 0.0)
    prob = prob / prob.sum(0)
    reached = torch.cumsum(prob, 0) > s["u"][:, :f].double()
    first = torch.where(reached.any(0), reached.int().argmax(0), ok.sum(0) - 1)
    return None, prob.gather(0, first[None])[0]
