"""A dense layer, the loss on top of one, and the clipping of gradients, as measurable cases.

DenseAffine: z = W x + b + residual, y = activation(z), and its backward pass.  LossDenseSoftmaxCrossEntropy: the cross entropy of softmax(W x + b) against
labels, with the gradients of x, W and b.  GradientNorm: the norm of a list of gradients, alone and with the Adam step that takes them clipped to a norm.

Frame buffers are node-major and frame-minor, as everywhere in this framework: [nodes, pitch] rows of fp32 frames or packed bits.  W is [outputs, inputs].
Each operator has its plain form (elementary torch operations in 32 bits) beside the framework's call.
"""
import math

import torch

own = False

LEARNING_RATE, BETA1, BETA2 = 0.001, 0.9, 0.999

ACTIVATIONS = ("none", "relu", "sigmoid", "hard_tanh")


# ---- what is measured ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one frame of a served network: latency
        {"name": "dense, one frame", "op": "dense", "inputs": 1024, "outputs": 1024, "frames": 1, "bits": False, "activation": "relu", "residual": True},
        # a small batch of requests behind a binary network, odd
        {"name": "dense, a few frames of packed bits", "op": "dense", "inputs": 6144, "outputs": 1024, "frames": 65, "bits": True, "activation": "hard_tanh", "residual": False},
        # the first layer of the classifier at its training batch
        {"name": "dense, a classifier's layer", "op": "dense", "inputs": 784, "outputs": 6144, "frames": 1024, "bits": False, "activation": "relu", "residual": False},
        # the headline layer's size, activations as a binary network leaves them, a shortcut beside them
        {"name": "dense over packed bits, large", "op": "dense", "inputs": 4096, "outputs": 4096, "frames": 8192, "bits": True, "activation": "none", "residual": True},
        # a training step at an odd batch
        {"name": "dense backward, odd sizes", "op": "dense_backward", "inputs": 1024, "outputs": 1001, "frames": 1000, "bits": False, "activation": "sigmoid", "residual": False},
        {"name": "dense backward, large", "op": "dense_backward", "inputs": 4096, "outputs": 4096, "frames": 8192, "bits": False, "activation": "relu", "residual": True},
        # the smallest training step: ten classes, 64 frames
        {"name": "cross entropy, ten classes", "op": "loss", "inputs": 1024, "channels": 10, "frames": 64, "bits": False, "gradients": True},
        {"name": "cross entropy, odd sizes", "op": "loss", "inputs": 777, "channels": 1001, "frames": 1000, "bits": False, "gradients": True},
        # evaluation: the loss alone, inputs from a binary network
        {"name": "cross entropy, evaluation", "op": "loss", "inputs": 1024, "channels": 10007, "frames": 513, "bits": True, "gradients": False},
        # a training step over many channels
        {"name": "cross entropy, many channels", "op": "loss", "inputs": 1024, "channels": 32768, "frames": 4096, "bits": False, "gradients": True},
        # the tables of the classifier 784-6144-1024-70 (64 entries a node) before its Adam step
        {"name": "gradient norm, a classifier's tables", "op": "norm", "tensors": 3, "values": (6144 + 1024 + 70) * 64, "share": 0.0, "step": False},
        # the weights and biases of a network of dense layers: the Adam step with clipped gradients
        {"name": "clipped step, large", "op": "norm", "tensors": 18, "values": 1 << 26, "share": 0.1, "step": True},
    ]


def _size(rng, lo, hi):
    """spread over the logarithm of the range"""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["dense", "dense_backward", "loss", "norm"])
    if op == "norm":
        step = rng.random() < 0.5
        tensors = _size(rng, 1, 18 if step else 300)
        return {"op": op, "tensors": tensors, "values": _size(rng, 64 * tensors, 1 << (26 if step else 28)), "share": round(rng.uniform(0.02, 1.5), 3) if step else 0.0, "step": step}
    inputs = _size(rng, 8, 8192)
    if op == "loss":
        channels = _size(rng, 2, 65536)
        frames = _size(rng, 1, max(1, min(8192, (1 << 37) // (inputs * channels))))
        return {"op": op, "inputs": inputs, "channels": channels, "frames": frames, "bits": rng.random() < 0.25, "gradients": rng.random() < 0.75}
    outputs = _size(rng, 2, 8192)
    frames = _size(rng, 1, max(1, min(16384, (1 << 37) // (inputs * outputs))))
    return {"op": op, "inputs": inputs, "outputs": outputs, "frames": frames, "bits": rng.random() < 0.3, "activation": rng.choice(ACTIVATIONS),
            "residual": rng.random() < 0.5}


def _pitch(frames):
    """floats from row to row, as the framework's buffers have them: whole 256 bytes, not a multiple of 2 KiB"""
    p = (frames + 63) // 64 * 64
    return p + 128 if p % 512 == 0 else p


def _words(frames):
    p = (frames + 2047) // 2048 * 64
    return p + 96 if p % 512 == 0 else p


def work(case):
    if case["op"] == "norm":
        n = case["values"]
        return {"bytes": (28 if case["step"] else 4) * n, "flops": (14 if case["step"] else 2) * n}
    i, f = case["inputs"], case["frames"]
    x = i * f / 8 if case["bits"] else 4 * i * f
    if case["op"] == "loss":
        c = case["channels"]
        if not case["gradients"]:
            return {"bytes": x + 4 * c * i + 4 * c + 12 * f, "flops": 2 * c * i * f}
        return {"bytes": x + 4 * i * f + 8 * c * i + 8 * c + 12 * f, "flops": 6 * c * i * f}
    o = case["outputs"]
    if case["op"] == "dense":
        return {"bytes": x + 4 * o * i + 4 * o + (8 if case["residual"] else 4) * o * f, "flops": 2 * o * i * f}
    reads = 4 if case["activation"] == "none" else 8
    return {"bytes": x + 4 * i * f + 8 * o * i + 4 * o + (reads + (4 if case["residual"] else 0)) * o * f, "flops": 4 * o * i * f}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------
def _rows(gen, nodes, frames, scale=1.0):
    """[nodes, pitch] frames; what lies behind a row's last frame is nobody's"""
    return torch.randn((nodes, _pitch(frames)), generator=gen, device="cuda").mul_(scale)


def _tensor_sizes(case):
    """sizes of many magnitudes, as weights and biases have them; they add up to the case's values"""
    n, total = case["tensors"], case["values"]
    if n == 3 and total == (6144 + 1024 + 70) * 64:
        return [6144 * 64, 1024 * 64, 70 * 64]
    share = [math.exp(-0.37 * (k * 7 % n) * 20.0 / n) for k in range(n)]
    sizes = [max(1, int((total - n) * s / sum(share))) for s in share]
    sizes[0] += total - sum(sizes)
    return sizes


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = dict(case)
    if case["op"] == "norm":
        state["grads"] = [torch.randn(n, generator=gen, device="cuda").mul_(10.0 ** (k % 5 - 3)) for k, n in enumerate(_tensor_sizes(case))]
        state["max_norm"] = math.inf
        if case["step"]:                         # in the middle of a training run; clipped to a share of the norm that the gradients have
            state["max_norm"] = case["share"] * math.sqrt(sum(float(g.double().square().sum()) for g in state["grads"]))
            state["params"] = [torch.randn(g.shape, generator=gen, device="cuda") for g in state["grads"]]
            state["m"] = [0.05 * torch.randn(g.shape, generator=gen, device="cuda") for g in state["grads"]]
            state["v"] = [0.01 * torch.rand(g.shape, generator=gen, device="cuda") for g in state["grads"]]
            state["t"] = 1
        return state
    f, i = case["frames"], case["inputs"]
    if case["bits"]:
        state["x"] = torch.randint(-(1 << 31), 1 << 31, (i, _words(f)), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    else:
        state["x"] = _rows(gen, i, f)
    o = case["channels"] if case["op"] == "loss" else case["outputs"]
    state["W"] = torch.randn((o, i), generator=gen, device="cuda").mul_((3.0 if case["op"] == "loss" else 1.0) / math.sqrt(i))
    state["b"] = torch.randn(o, generator=gen, device="cuda").mul_(0.1)
    if case["op"] == "loss":
        label = torch.randint(0, o, (1, _pitch(f)), generator=gen, device="cuda", dtype=torch.int32)
        weight = torch.rand((1, _pitch(f)), generator=gen, device="cuda") + 0.5
        label[:, 4::9] = -1                       # frames without a label, and padding of the batch
        weight[:, 7::8] = 0.0
        state["label"], state["weight"] = label, weight
        state["weight_sum"] = float(torch.where(label >= 0, weight, 0.0)[:, :f].double().sum())
        return state
    if case["op"] == "dense":
        state["r"] = _rows(gen, o, f) if case["residual"] else None
        return state
    state["dy"] = _rows(gen, o, f)
    state["y"] = None
    if case["activation"] != "none":              # the forward pass's output
        state["y"] = _activated(_rows(gen, o, f), case["activation"])
    return state


def _activated(z, activation):
    if activation == "relu":
        return torch.clamp(z, min=0.0)
    if activation == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    if activation == "hard_tanh":
        return torch.clamp(z, -1.0, 1.0)
    return z


def _slope(y, activation):
    """the activation's derivative, from its value"""
    if activation == "relu":
        return (y > 0).to(y.dtype)
    if activation == "sigmoid":
        return y * (1.0 - y)
    if activation == "hard_tanh":
        return ((y > -1.0) & (y < 1.0)).to(y.dtype)
    return torch.ones_like(y)


def _values(s):
    """x as fp32 [inputs, frames]"""
    x, f = s["x"], s["frames"]
    if not s["bits"]:
        return x[:, :f]
    bit = torch.arange(32, device=x.device, dtype=torch.int32)
    return ((x[:, :(f + 31) // 32, None] >> bit) & 1).reshape(x.shape[0], -1)[:, :f].float()


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(state):
    return {"dense": _dense, "dense_backward": _dense_backward, "loss": _loss, "norm": _norm}[state["op"]](state)


def _dense(s):
    f = s["frames"]
    if own:
        from binarybrain_amd import ops
        if s["bits"]:
            y = ops.bit_dense_affine_forward(s["x"], s["W"], s["b"], f, _pitch(f), activation=s["activation"], residual=s["r"])
        else:
            y = ops.dense_affine_forward(s["x"], s["W"], s["b"], f, activation=s["activation"], residual=s["r"])
        return y[:, :f]
    z = s["W"] @ _values(s) + s["b"][:, None]
    if s["r"] is not None:
        z = z + s["r"][:, :f]
    return _activated(z, s["activation"])


def _dense_backward(s):
    f = s["frames"]
    if own:
        from binarybrain_amd import ops
        call = ops.bit_dense_affine_backward if s["bits"] else ops.dense_affine_backward
        dx, dW, db, dr = call(s["x"], s["dy"], s["W"], f, activation=s["activation"], y=s["y"], want_dr=s["residual"])
        return (dx[:, :f], dW, db) + ((dr[:, :f],) if s["residual"] else ())
    dz = s["dy"][:, :f]
    if s["y"] is not None:
        dz = dz * _slope(s["y"][:, :f], s["activation"])
    return (s["W"].t() @ dz, dz @ _values(s).t(), dz.sum(1)) + ((dz,) if s["residual"] else ())


def _loss(s):
    f = s["frames"]
    if own:
        from binarybrain_amd import ops
        if s["bits"]:
            loss, dx, dW, db = ops.bit_loss_dense_softmax_cross_entropy(s["x"], s["W"], s["b"], s["label"], f, _pitch(f), weight=s["weight"], weight_sum=s["weight_sum"],
                                                                        want_gradients=s["gradients"])
        else:
            loss, dx, dW, db = ops.loss_dense_softmax_cross_entropy(s["x"], s["W"], s["b"], s["label"], f, weight=s["weight"], weight_sum=s["weight_sum"],
                                                                    want_gradients=s["gradients"])
        loss = loss[None, :, :f]
        return (loss, dx[:, :f], dW, db) if s["gradients"] else loss
    x, label = _values(s), s["label"][0, :f].long()
    counts = (label >= 0) & (label < s["channels"])
    w = torch.where(counts, s["weight"][0, :f], 0.0)
    at = torch.where(counts, label, 0)[None]
    z = s["W"] @ x + s["b"][:, None]
    z = z - z.amax(0)
    e = torch.exp(z)
    total = e.sum(0)
    loss = w * (torch.log(total) - z.gather(0, at))
    if not s["gradients"]:
        return loss[None]
    # (a mean over no frames at all has no gradient)
    g = w / s["weight_sum"] if s["weight_sum"] > 0 else torch.zeros_like(w)
    dz = (e * (g / total)).scatter_add(0, at, -g[None])
    return loss[None], s["W"].t() @ dz, dz @ x.t(), dz.sum(1)


def _norm(s):
    if own:
        return _norm_own(s)
    grads = s["grads"]
    norm = torch.sqrt(torch.stack([g.square().sum() for g in grads]).sum())
    scale = torch.clamp(s["max_norm"] / norm, max=1.0)
    both = torch.stack([norm, scale])
    if not s["step"]:
        return both
    rate = LEARNING_RATE * math.sqrt(1.0 - BETA2 ** s["t"]) / (1.0 - BETA1 ** s["t"])
    s["t"] += 1
    p, m, v = s["params"], s["m"], s["v"]
    g = torch._foreach_mul(grads, scale)
    torch._foreach_add_(m, torch._foreach_sub(g, m), alpha=1.0 - BETA1)
    torch._foreach_add_(v, torch._foreach_sub(torch._foreach_mul(g, g), v), alpha=1.0 - BETA2)
    torch._foreach_sub_(p, torch._foreach_div(torch._foreach_mul(m, rate), torch._foreach_add(torch._foreach_sqrt(v), 1.0e-7)))
    return both, p, m, v


def _norm_own(s):
    from binarybrain_amd import ops
    if not s["step"]:
        if "table" not in s:                     # a program has it beside its gradients, as long as these stay where they are
            s["table"] = ops.GradientTable(s["grads"])
        return s["table"].norm()
    if "adam" not in s:
        s["adam"] = ops.AdamState(s["params"], s["grads"], LEARNING_RATE, BETA1, BETA2, m=s["m"], v=s["v"])
    return s["adam"].step(max_norm=s["max_norm"]), s["params"], s["m"], s["v"]


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        total = sum(float(torch.dot(g.double(), g.double())) for g in s["grads"])
        norm = total ** 0.5
        scale = 1.0 if norm <= s["max_norm"] else s["max_norm"] / norm
        both = torch.tensor([norm, scale], dtype=torch.float64)
        if not case["step"]:
            return both
        rate = LEARNING_RATE * (1.0 - BETA2) ** 0.5 / (1.0 - BETA1)
        m = [a.double() * BETA1 + g.double() * (scale * (1.0 - BETA1)) for a, g in zip(s["m"], s["grads"])]
        v = [a.double() * BETA2 + (g.double() * scale) ** 2 * (1.0 - BETA2) for a, g in zip(s["v"], s["grads"])]
        return both, [a.double() - rate * b / (c.sqrt() + 1.0e-7) for a, b, c in zip(s["params"], m, v)], m, v
    f = case["frames"]
    if case["bits"]:
        shift = torch.arange(f, device="cuda")
        x = ((s["x"].long()[:, shift // 32] >> (shift % 32)) & 1).double()
    else:
        x = s["x"][:, :f].double()
    W, b = s["W"].double(), s["b"].double()
    if case["op"] == "dense":
        z = torch.addmm(b[:, None].expand(-1, f) + (s["r"][:, :f].double() if case["residual"] else 0.0), W, x)
        return {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, 0.0), "sigmoid": lambda: torch.sigmoid(z), "hard_tanh": lambda: z.clip(-1, 1)}[case["activation"]]()
    if case["op"] == "dense_backward":
        dz = s["dy"][:, :f].double()
        if case["activation"] != "none":
            y = s["y"][:, :f].double()
            dz = dz * {"relu": lambda: y > 0, "sigmoid": lambda: y - y * y, "hard_tanh": lambda: y.abs() < 1}[case["activation"]]()
        out = torch.mm(W.T, dz), torch.mm(dz, x.T), dz.sum(dim=1)
        return out + ((dz,) if case["residual"] else ())
    label, w = s["label"][0, :f].long(), s["weight"][0, :f].double()
    w = w * (label >= 0)
    log_p = torch.log_softmax(torch.addmm(b[:, None], W, x), dim=0)
    there = label.clamp_min(0)
    loss = -w * log_p[there, torch.arange(f, device="cuda")]
    if not case["gradients"]:
        return loss[None]
    dz = log_p.exp_()
    dz[there, torch.arange(f, device="cuda")] -= 1.0
    dz *= w / s["weight_sum"] if s["weight_sum"] else 0.0
    return loss[None], W.T @ dz, dz @ x.T, dz.sum(dim=1)
