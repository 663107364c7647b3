"""What the vocabulary operators are timed on: the softmax cross entropy of a last layer with a large vocabulary, taken in
pieces of the vocabulary without keeping the logits, and the distillation from a teacher's top logits over the same layer;
each as the loss alone and as a training step's loss, error and weight gradient.

Everything but the loss is integer arithmetic with a fixed definition (``_exp_weights`` and what follows it), so whole-number
outputs are the same bit for bit whatever computes them; an int8 error comes with its exponent, both as the whole numbers
that they are.
"""
import math

import torch

own = False

PIECE = 64  # vocabulary entries whose exponentials are summed relative to their own maximum
NEAREST, STOCHASTIC, PSEUDO = "nearest", "stochastic", "pseudo"


def listed():
    return [
        # scoring one token: a small vocabulary, where the launches count, and a large one, where the weights' bytes do
        _case("loss 1x512x1000", "loss", 1, 512, 1000),
        _case("loss 1x2048x131072", "loss", 1, 2048, 131072),
        # the likelihood of a batch of short texts, sizes that are nobody's multiple, a third of the rows padding
        _case("loss 1023x776x50021", "loss", 1023, 776, 50021, ignored=0.33),
        # a validation pass over a long text
        _case("loss 8192x1024x32768", "loss", 8192, 1024, 32768),
        # training steps: a small model's few tokens, an ordinary batch in each rounding, a ragged one, the largest
        _case("train 48x256x4096", "train", 48, 256, 4096),
        _case("train 2048x1024x32768", "train", 2048, 1024, 32768),
        _case("train 1500x520x32001 stochastic", "train", 1500, 520, 32001, rounding=STOCHASTIC, ignored=0.2),
        _case("train 777x1000x10007 nearest", "train", 777, 1000, 10007, rounding=NEAREST, ignored=0.1),
        _case("train 8192x2048x65536", "train", 8192, 2048, 65536),
        # scoring a student against a teacher's sixteen best; training on thirty-two of them; ragged lists at a temperature
        _case("distill loss 512x1024x32768", "distill_loss", 512, 1024, 32768, top=16),
        _case("distill train 4096x1024x32768", "distill_train", 4096, 1024, 32768, top=32),
        _case("distill train 333x640x20011", "distill_train", 333, 640, 20011, top=50, top_type="int32", ragged=True, temperature=1),
    ]


def _case(name, kind, tokens, features, vocab, rounding=PSEUDO, ignored=0.0, top=0, top_type="int8", ragged=False, temperature=0):
    c = {"kind": kind, "tokens": tokens, "features": features, "vocab": vocab, "rounding": rounding, "ignored": ignored,
         "top": top, "top_type": top_type, "ragged": ragged, "temperature": temperature}
    return {"name": name, **c} if name else c


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("loss", "train", "train", "distill_loss", "distill_train"))
    features = _log_int(rng, 64, 2048)
    if rng.random() < 0.7:  # most layers are multiples of 16 wide
        features = max(64, features // 16 * 16)
    vocab = _log_int(rng, 500, 131072)
    tokens = _log_int(rng, 1, max(1, min(8192, (1 << 27) // vocab)))
    distill = kind.startswith("distill")
    return _case(None, kind, tokens, features, vocab, rounding=rng.choice((PSEUDO, PSEUDO, NEAREST, STOCHASTIC)),
                 ignored=0.0 if distill else rng.choice((0.0, 0.1, 0.5)), top=_log_int(rng, 1, 64) if distill else 0,
                 top_type=rng.choice(("int8", "int32")), ragged=rng.random() < 0.5, temperature=rng.choice((0, 0, 1, 2)) if distill else 0)


def prepare(case, seed):
    """A last layer in training: features and weights of a normal distribution in int8, exponents that put the logits' spread
    at about 2.5, the wanted entry's logit from nowhere to far above the others; the teacher's best entries start at the
    wanted one."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    T, F, V = case["tokens"], case["features"], case["vocab"]
    w = (torch.randn(V, F, device=dev, generator=g) * 30).round_().clamp_(-127, 127).to(torch.int8)
    target = torch.randint(0, V, (T,), device=dev, generator=g)
    lift = torch.rand(T, 1, device=dev, generator=g) * (4.8 / math.sqrt(F))
    x = torch.randn(T, F, device=dev, generator=g) * 24 + lift * w[target].float()
    x = x.round_().clamp_(-127, 127).to(torch.int8)
    e = round(math.log2(2.5 / (math.sqrt(F) * 720)))
    word = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = {"case": dict(case), "x": x, "w": w, "exp_x": word(e + 9), "exp_w": word(-9),
         "seed": torch.randint(0, 1 << 62, (1,), device=dev, generator=g)}
    if case["top"]:
        K = case["top"]
        index = torch.randint(0, V, (T, K), device=dev, generator=g)
        index[:, 0] = target
        if case["ragged"]:  # lists of any length, the empty one among them
            count = torch.randint(0, K + 1, (T, 1), device=dev, generator=g)
            index = torch.where(torch.arange(K, device=dev) < count, index, -1)
        top = (torch.randn(T, K, device=dev, generator=g) * 25 + 60).sort(1, descending=True).values.round_().clamp_(-127, 127)
        wide = case["top_type"] == "int32"
        s.update(index=index, top=(top * 1000 if wide else top).to(torch.int32 if wide else torch.int8), exp_top=word(-13 if wide else -4))
    else:
        s["target"] = torch.where(torch.rand(T, device=dev, generator=g) < case["ignored"], -100, target)
    return s


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    e = s["exp_x"] + s["exp_w"] - c["temperature"]
    acc = _product(s["x"], s["w"].t())
    M, S = _row_statistics(acc, e)
    if c["top"]:
        entries = s["index"]
        share, teacher = _teacher(s["top"], entries >= 0, s["exp_top"] - c["temperature"])
        scale = 4.0 ** c["temperature"]
    else:
        entries = torch.where(s["target"] == -100, -1, s["target"]).unsqueeze(1)
        share, teacher, scale = entries.clamp(max=0) + 1, 0.0, 1.0
    used, at = entries >= 0, entries.clamp(min=0)
    unit = torch.exp2(e.double())
    # -log p of each entry, weighted, and q log q of the teacher
    far = (M - acc.gather(1, at)) * unit + torch.log(S.double() / 2.0 ** 34)
    weight = share.double() / share.sum(1, keepdim=True).clamp(min=1)
    loss = (scale * ((weight * far).sum(1) + teacher)).where(used.any(1), 0.0).float()
    if c["kind"].endswith("loss"):
        return loss

    # the error of the logits, in units of 2^-30, narrowed to 2^-7
    n = torch.frexp(S.double()).exponent.long() - 32
    p = ((_exp_weights(M - acc, e) * (((1 << 63) - 1) // (S >> n))) >> 32) >> (n - 3)
    p = p * used.any(1, keepdim=True)
    p.scatter_add_(1, at, -((share << 30) // share.sum(1, keepdim=True).clamp(min=1)) * used)
    four = (c["vocab"] + 3) // 4 * 4
    rnd = _random_words(s["seed"], 0xFFFF, c["tokens"], four)[:, :c["vocab"]] if c["rounding"] == STOCHASTIC else None
    err = _narrow(p, torch.full((), 23, dtype=torch.int64, device=p.device), c["rounding"], rnd)
    # back to the features and the weights
    e32, g32 = _product(err, s["w"]), _product(err.t(), s["x"])
    top = e32.abs().amax()
    shift = (torch.frexp((top - 1).clamp(min=0).double()).exponent.long() - 7).clamp(min=0)
    mode = STOCHASTIC if c["rounding"] == STOCHASTIC else NEAREST
    words = None
    if mode == STOCHASTIC:
        pad = -e32.numel() % 4
        words = _random_words(s["seed"], 1, 1, e32.numel() + pad)[0, :e32.numel()].view_as(e32)
    e8 = _narrow(e32, shift, mode, words)
    return loss, e8.to(torch.int8), (shift + s["exp_w"] - 7 + c["temperature"]).to(torch.int32), g32.to(torch.int32), g32.abs().amax().to(torch.int32).reshape(1)


def _run_own(s):
    from niti_b200 import ops
    c = s["case"]
    layer = (s["x"], s["exp_x"], s["w"], s["exp_w"])
    if c["kind"] == "loss":
        return ops.vocab_loss(*layer, s["target"])
    if c["kind"] == "distill_loss":
        return ops.vocab_distill_loss(*layer, s["index"], s["top"], s["exp_top"], c["temperature"])
    loss_mode = {NEAREST: ops.ROUND_NEAREST, STOCHASTIC: ops.ROUND_STOCHASTIC, PSEUDO: ops.ROUND_PSEUDO_STOCHASTIC}[c["rounding"]]
    err_mode = ops.ROUND_STOCHASTIC if c["rounding"] == STOCHASTIC else ops.ROUND_NEAREST
    how = dict(loss_mode=loss_mode, err_mode=err_mode, seed=s["seed"], loss_stream=0xFFFF, err_stream=1)
    if c["kind"] == "train":
        return ops.vocab_train(*layer, s["target"], **how)
    return ops.vocab_distill_train(*layer, s["index"], s["top"], s["exp_top"], c["temperature"], **how)


def _product(a, b):
    """The exact product of whole numbers: in 64 bits every sum of this size is exact."""
    return (a.double() @ b.double()).long()


def _exp_weights(d, e):
    """E(d) = 2^30 exp(-d 2^e) for whole d >= 0, in fixed point: u is d 2^e log2(e) in units of 2^-25 plus a half, 2^-phi for its
    fraction less a half comes from a quartic (largest relative error 2.9e-6), its whole part is a shift to the right.  From D
    on (31 powers of two) the result is 0."""
    e = e.long().clamp(max=5)
    D = torch.where(e < 0, 43 << (-e - 1).clamp(0, 26), 21 + (1 << e.clamp(min=0)) >> e.clamp(min=0))
    D = torch.where(e <= -28, (1 << 32) - 1, D)
    u = ((torch.minimum(d, D) << (e + 26).clamp(0, 31)) * (0xB8AA3B29 >> (-26 - e).clamp(0, 63)) >> 32) + (1 << 24)
    phi = ((u & ((1 << 25) - 1)) - (1 << 24)) << 7
    q = (phi * 10289510 >> 32) - 60029066
    q = (phi * q >> 32) + 257956795
    q = (phi * q >> 32) - 744236436
    return ((phi * q >> 32) + (1 << 30)) >> (u >> 25)


def _row_statistics(acc, e):
    """Each row's maximum and its sum of exponentials relative to it (1.0 = 2^34), [T, 1] both: in pieces, each relative to
    its own maximum first."""
    T, V = acc.shape
    low = -1 << 40
    pieces = torch.nn.functional.pad(acc, (0, -V % PIECE), value=low).view(T, -1, PIECE)
    m = pieces.amax(2)
    part = _exp_weights(m.unsqueeze(2) - pieces, e).masked_fill_(pieces == low, 0).sum(2) >> 6
    M = m.amax(1, keepdim=True)
    return M, (part * _exp_weights(M - m, e) >> 20).sum(1, keepdim=True)


def _teacher(top, used, e):
    """The teacher's shares in units that sum to anything, and sum q log q of each row."""
    top = top.long()
    best = top.masked_fill(~used, -1 << 40).amax(1, keepdim=True)
    d = (best - top).where(used, 0)
    share = _exp_weights(d, e) * used
    total = share.sum(1, keepdim=True).clamp(min=1).double()
    logq = -d * torch.exp2(e.double()) - torch.log(total / 2.0 ** 30)
    return share, (share / total * logq).sum(1)


def _narrow(v, shift, mode, rnd):
    """A right shift of whole numbers to +-127, rounded; without a shift the low byte, as a cast to int8 gives it."""
    a = v.abs()
    lo = a & ((1 << shift) - 1)
    if mode == NEAREST:
        up = lo >> (shift - 1).clamp(min=0)
    elif mode == STOCHASTIC:
        up = lo > (rnd & ((1 << shift) - 1))
    else:
        h = shift >> 1
        up = (lo >> h) > ((lo & ((1 << h) - 1)) << (shift & 1))
    y = ((a >> shift) + up).clamp(max=127) * v.sign()
    return torch.where(shift > 0, y, v)


def _random_words(seed, stream, rows, columns):
    """The words of elements 0, 1, ... of a stream: Philox4x32-10 keyed by the seed, four words to a counter."""
    block = torch.arange(rows * columns // 4, device=seed.device)
    low = 0xFFFFFFFF
    c = [block & low, block >> 32, torch.full_like(block, stream), torch.zeros_like(block)]
    k = [seed & low, seed >> 32 & low]
    for _ in range(10):
        (h0, l0), (h1, l1) = _wide(c[0], 0xD2511F53), _wide(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k[0], l1, h0 ^ c[3] ^ k[1], l0]
        k = [k[0] + 0x9E3779B9 & low, k[1] + 0xBB67AE85 & low]
    return torch.stack(c, 1).view(rows, columns)


def _wide(a, m):
    """High and low word of a 32 x 32 bit product, both factors below 2^32."""
    lo = a * (m & 0xFFFF)
    hi = a * (m >> 16) + (lo >> 16)
    return hi >> 16, (hi << 16 | lo & 0xFFFF) & 0xFFFFFFFF


def work(case):
    """Operands in once, results out once; the logits' product, and for training the two that lead back."""
    T, F, V = case["tokens"], case["features"], case["vocab"]
    train = case["kind"].endswith("train")
    size = T * F + V * F + 12 * T + 12 * T * case["top"]
    return {"bytes": size + (T * F + 4 * V * F if train else 0), "flops": (6 if train else 2) * T * V * F}


def exact(case, seed):
    """The loss by its definition in 64 bits: a softmax of the dequantised logits with the library's exponential.  The whole
    numbers beside it (error, exponent, gradient) are defined by integer arithmetic and have no other value."""
    s = prepare(case, seed)
    t = 2.0 ** case["temperature"]
    logits = s["x"].double() @ s["w"].double().t()
    logp = torch.log_softmax(logits * (2.0 ** float(s["exp_x"] + s["exp_w"]) / t), 1)
    if case["top"]:
        used = s["index"] >= 0
        z = (s["top"].double() * (2.0 ** float(s["exp_top"]) / t)).masked_fill(~used, -math.inf)
        logq = torch.log_softmax(z, 1)
        terms = logq.exp() * (logq - logp.gather(1, s["index"].clamp(min=0)))
        loss = t * t * terms.where(used, 0.0).sum(1)
    else:
        used = s["target"] >= 0
        loss = (-logp.gather(1, s["target"].clamp(min=0).unsqueeze(1)).squeeze(1)).where(used, 0.0)
    return loss if case["kind"].endswith("loss") else (loss, None, None, None, None)
