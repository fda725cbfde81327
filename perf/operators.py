"""The operators of a transformer's feed-forward block, as cases to time: the gated block in 16 bits (one token, prompts, training and its
backward pass), matrix-vector products with 4-bit weights and group scales, the gated block on 4-bit weights, and the quantisation that
brings weights into that form.

A case is a dict of plain values; "op" names the operator.  prepare() makes the operands of one case on the GPU, run() makes one pass:
with `own` the calls a program makes of this library, without it the same in elementary torch operations in 32 bits.  exact() is the
definition in 64 bits.

4-bit weights W[n][k] = scale[n][k / group] * v, v in -8..7, are held in one buffer.  A tile of 16 rows x 128 columns takes 1024 bytes; tiles
run along k first.  In a tile 16-byte unit 16 * (k % 32 / 8) + n % 16 holds in word k % 128 / 32 the eight columns k % 8 = e, v + 8 at bit
4 * (e / 2) + 16 * (e % 2).  Behind the tiles lie the scales, [tile rows][tile columns][16][128 / group]; rows and columns that fill up the
last tiles hold v = 0 and scale 0.
"""
import math

import torch

own = False
DEVICE = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


# ---- the cases --------------------------------------------------------------------------------------------------------

def listed():
    return [
        # A single token through a block whose weights stay in 16 bits: their bytes.
        dict(name="ffn_token_bf16", op="ffn", type="bf16", rows=1, d=2048, f=8192, act="silu", save=False),
        # A prompt, or a batch of them: the matrix cores.
        dict(name="ffn_prompt_fp16", op="ffn", type="fp16", rows=4096, d=2048, f=8192, act="gelu_tanh", save=False),
        # The forward pass of a training step on odd sizes: pre-activations are kept, no row begins on a whole word of 16 bytes.
        dict(name="ffn_train_ragged_bf16", op="ffn", type="bf16", rows=777, d=1111, f=2731, act="silu", save=True),
        # The backward pass of a training step: the largest work here.
        dict(name="ffn_backward_bf16", op="ffn_backward", type="bf16", rows=4096, d=2048, f=8192, act="silu"),
        # The same on a short, ragged sequence.
        dict(name="ffn_backward_ragged_fp16", op="ffn_backward", type="fp16", rows=509, d=722, f=1930, act="gelu"),
        # The smallest call: launch and host time are all there is.
        dict(name="matvec_small_fp16", op="matvec", type="fp16", rows=1, k=512, n=512, group=32, gap=0),
        # A projection for a single token.
        dict(name="matvec_token_fp16", op="matvec", type="fp16", rows=1, k=4096, n=4096, group=128, gap=0),
        # A step of several sequences at once, sizes that fill no tile, rows that lie apart.
        dict(name="matvec_ragged_bf16", op="matvec", type="bf16", rows=13, k=4111, n=12001, group=64, gap=9),
        # The block for a single token on 4-bit weights, at the size of a large model: more than the caches hold.
        dict(name="ffn_int4_token_bf16", op="ffn_int4", type="bf16", rows=1, d=8192, f=32768, group=128, act="silu", gap=0),
        # The same for a batch of sequences on a smaller one.
        dict(name="ffn_int4_batch_fp16", op="ffn_int4", type="fp16", rows=33, d=2048, f=5500, group=32, act="gelu", gap=0),
        # Weights into 4 bits and back, as a program that quantises a checkpoint and looks at the error does.
        dict(name="quantize_bf16", op="quantize", type="bf16", n=16384, k=4096, group=128),
        dict(name="quantize_ragged_fp16", op="quantize", type="fp16", n=1001, k=1111, group=32),
    ]


def _log(rng, lo, hi):
    """an integer spread over the logarithm of [lo, hi]"""
    v = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return v + 1 if v == 3072 else v


def _width(rng, lo, hi):
    """a feature count: most are multiples of 8 or 64, some are odd"""
    v, step = _log(rng, lo, hi), rng.choice((1, 1, 8, 64, 64))
    v = max(lo, min(hi, (v + step - 1) // step * step))
    return v + step if v == 3072 else v


def _drawn(rng):
    op, t = rng.choice(("ffn", "ffn", "ffn_backward", "matvec", "matvec", "ffn_int4", "quantize")), rng.choice(("fp16", "bf16"))
    case = dict(op=op, type=t)
    if op in ("ffn", "ffn_backward"):
        case.update(rows=_log(rng, 1, 8192), d=_width(rng, 64, 8192), f=_width(rng, 64, 32768), act=rng.choice(ACTS))
        if op == "ffn":
            case["save"] = rng.random() < 0.4
        return case
    group = rng.choice((32, 64, 128))
    if op == "quantize":
        return dict(case, n=_width(rng, 64, 32768), k=_width(rng, 64, 8192), group=group)
    case.update(rows=_log(rng, 1, 64), group=group, gap=rng.choice((0, 0, 8, 3)))
    if op == "matvec":
        return dict(case, k=_width(rng, 64, 32768), n=_width(rng, 64, 32768))
    return dict(case, d=_width(rng, 64, 8192), f=_width(rng, 64, 32768), act=rng.choice(ACTS))


# the most operations and bytes of a drawn case of each kind: no more than the largest listed one's
_MOST = {"ffn": (2.7e11, 3.0e8), "ffn_backward": (5.4e11, 4.0e8), "matvec": (1e11, 2.9e8), "ffn_int4": (1e11, 2.9e8), "quantize": (1e11, 3.4e8)}


def draw(rng):
    while True:
        case = _drawn(rng)
        w = work(case)
        if w["flops"] <= _MOST[case["op"]][0] and w["bytes"] <= _MOST[case["op"]][1]:
            return case


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def _packed_bytes(n, k, group):
    """values and scales of an n x k matrix"""
    return n * k // 2 + 2 * n * -(-k // group)


def work(case):
    """Multiply-adds count as two operations; every input is read once and every output written once."""
    op = case["op"]
    if op in ("ffn", "ffn_backward"):
        m, d, f = case["rows"], case["d"], case["f"]
        if op == "ffn":
            return dict(bytes=2 * (m * d + 2 * f * d + (3 if case["save"] else 1) * m * f), flops=4 * m * d * f)
        return dict(bytes=2 * (2 * m * d + 4 * f * d + 3 * m * f), flops=8 * m * d * f)
    if op == "matvec":
        m, k, n = case["rows"], case["k"], case["n"]
        return dict(bytes=_packed_bytes(n, k, case["group"]) + 2 * m * (k + n), flops=2 * m * n * k)
    if op == "ffn_int4":
        m, d, f = case["rows"], case["d"], case["f"]
        return dict(bytes=2 * _packed_bytes(f, d, case["group"]) + 2 * m * (d + f), flops=4 * m * d * f)
    n, k = case["n"], case["k"]
    return dict(bytes=2 * (2 * n * k + _packed_bytes(n, k, case["group"])), flops=4 * n * k)


# ---- operands ---------------------------------------------------------------------------------------------------------

class _Operands:
    """Seeded operands on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device=DEVICE)
        self.gen.manual_seed(seed)

    def normal(self, std, shape, dtype):
        return (torch.randn(shape, generator=self.gen, device=DEVICE) * std).to(dtype)

    def activations(self, rows, width, gap, dtype):
        """normed activations with the few large channels that they have, rows `gap` elements further apart than they are long"""
        x = torch.randn((rows, width + gap), generator=self.gen, device=DEVICE)
        large = torch.rand((width + gap,), generator=self.gen, device=DEVICE) < 0.004
        return (x * torch.where(large, 12.0, 1.0)).to(dtype)[:, :width]

    def packed(self, n, k, group, dtype):
        """normal weights of an n x k matrix in 4 bits"""
        w = torch.randn((n, k), generator=self.gen, device=DEVICE) / math.sqrt(k)
        return _pack(*_quantized(w.to(dtype), group), k, group)


def _quantized(w, group):
    """values (float) [n][columns, filled up to whole groups] and scales [n][groups] of 16-bit weights"""
    n, k = w.shape
    g = torch.nn.functional.pad(w.float(), (0, -k % group)).view(n, -1, group)
    scale = (g.abs().amax(-1) / 7).to(w.dtype)
    v = torch.round(g / scale.float().unsqueeze(-1)).nan_to_num(0.0).clamp(-7, 7)
    return v.view(n, -1), scale


def _pack(v, scale, k, group):
    n, tiles_n, tiles_k = v.shape[0], -(-v.shape[0] // 16), -(-k // 128)
    u = torch.nn.functional.pad(v.to(torch.int32) + 8, (0, tiles_k * 128 - v.shape[1], 0, tiles_n * 16 - n), value=8)
    # [row tile][row][column tile][word][quarter][pair][half] -> [row tile][column tile][quarter][row][word], pairs and halves summed
    u = u.view(tiles_n, 16, tiles_k, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 5, 6).to(torch.uint8)
    u = u[..., 0::2, :] | u[..., 1::2, :] << 4    # pairs 0, 1 and 2, 3 of a half word are one byte each
    values = u.transpose(-1, -2).reshape(-1)
    per_tile = 128 // group
    s = torch.nn.functional.pad(scale, (0, tiles_k * per_tile - scale.shape[1], 0, tiles_n * 16 - n))
    s = s.view(tiles_n, 16, tiles_k, per_tile).transpose(1, 2).reshape(-1)
    return torch.cat((values, s.contiguous().view(torch.uint8)))


def _unpack(packed, n, k, group, dtype):
    """the weights as floats"""
    tiles_n, tiles_k = -(-n // 16), -(-k // 128)
    u = packed[: tiles_n * tiles_k * 1024].view(tiles_n, tiles_k, 4, 16, 4, 2, 2, 1)
    u = torch.cat((u & 15, u >> 4), -1)    # [..., word, half, byte of it, nibble]
    v = u.view(tiles_n, tiles_k, 4, 16, 4, 2, 4).permute(0, 3, 1, 4, 2, 6, 5).reshape(tiles_n * 16, tiles_k * 128).float() - 8
    s = packed[tiles_n * tiles_k * 1024:].view(dtype).view(tiles_n, tiles_k, 16, 128 // group).transpose(1, 2).reshape(tiles_n * 16, -1, 1).float()
    return (v.view(tiles_n * 16, -1, group) * s).view(tiles_n * 16, -1)[:n, :k]


def prepare(case, seed):
    ops, op, t = _Operands(seed), case["op"], TYPES[case["type"]]
    state = dict(case=case, type=t)
    if op in ("ffn", "ffn_backward"):
        m, d, f = case["rows"], case["d"], case["f"]
        state["x"] = ops.activations(m, d, 0, t)
        state["gate"], state["up"] = (ops.normal(1 / math.sqrt(d), (f, d), t) for _ in range(2))
        if op == "ffn_backward":
            state["g"], state["u"] = ((state["x"].float() @ state[w].float().t()).to(t) for w in ("gate", "up"))
            state["dh"] = ops.normal(0.1, (m, f), t)
    elif op == "matvec":
        state["x"] = ops.activations(case["rows"], case["k"], case["gap"], t)
        state["w"] = ops.packed(case["n"], case["k"], case["group"], t)
    elif op == "ffn_int4":
        state["x"] = ops.activations(case["rows"], case["d"], case["gap"], t)
        state["gate"], state["up"] = (ops.packed(case["f"], case["d"], case["group"], t) for _ in range(2))
    else:
        state["w"] = ops.normal(0.02, (case["n"], case["k"]), t)
    return state


# ---- one pass, in the plain form ---------------------------------------------------------------------------------------

def _act(name, g):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    if name == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    if name == "relu":
        return g.clamp_min(0)
    return 1 / (1 + torch.exp(-g))


def _act_slope(name, g):
    if name in ("silu", "sigmoid"):
        s = 1 / (1 + torch.exp(-g))
        return s * (1 + g * (1 - s)) if name == "silu" else s * (1 - s)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) * math.sqrt(0.5 / math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    return (g > 0).to(g.dtype)


def _plain(state):
    case, t = state["case"], state["type"]
    op, act = case["op"], case.get("act")
    if op == "ffn":
        x = state["x"].float()
        g, u = x @ state["gate"].float().t(), x @ state["up"].float().t()
        h = (_act(act, g) * u).to(t)
        return dict(h=h, g=g.to(t), u=u.to(t)) if case["save"] else dict(h=h)
    if op == "ffn_backward":
        x, g, u, dh = (state[n].float() for n in ("x", "g", "u", "dh"))
        dg, du = dh * u * _act_slope(act, g), dh * _act(act, g)
        return dict(dx=(dg @ state["gate"].float() + du @ state["up"].float()).to(t), dgate=(dg.t() @ x).to(t), dup=(du.t() @ x).to(t))
    if op == "matvec":
        w = _unpack(state["w"], case["n"], case["k"], case["group"], t)
        return dict(y=(state["x"].float() @ w.t()).to(t))
    if op == "ffn_int4":
        x = state["x"].float()
        g, u = (x @ _unpack(state[w], case["f"], case["d"], case["group"], t).t() for w in ("gate", "up"))
        return dict(h=(_act(act, g) * u).to(t))
    n, k, group = case["n"], case["k"], case["group"]
    v, s = _quantized(state["w"], group)
    return dict(w=(v.view(n, -1, group) * s.float().unsqueeze(-1)).view(n, -1)[:, :k].to(t))


# ---- one pass, as a program calls the library ---------------------------------------------------------------------------

_context = None


def _library():
    """The process's library context, on the stream torch works on."""
    global _context
    if _context is None:
        from reference_model_amd import Context
        _context = Context(0)
        _context.set_stream(torch.cuda.current_stream().cuda_stream)
    return _context


def _calls(state):
    """The descriptors, result tensors and calls of a program that has these operands."""
    from reference_model_amd import capi
    ctx, case, t = _library(), state["case"], state["type"]
    op, dtype = case["op"], capi.FP16 if t == torch.float16 else capi.BF16
    act = {"silu": capi.ACT_SILU, "gelu": capi.ACT_GELU, "gelu_tanh": capi.ACT_GELU_TANH, "relu": capi.ACT_RELU,
           "sigmoid": capi.ACT_SIGMOID}[case.get("act", "silu")]
    empty = lambda *shape: torch.empty(shape, dtype=t, device=DEVICE)  # noqa: E731
    if op in ("ffn", "ffn_backward"):
        m, d, f = case["rows"], case["d"], case["f"]
        desc = ctx.gated_ffn_desc(dtype, act, m, d, f)
        if op == "ffn":
            out = dict(h=empty(m, f), g=empty(m, f), u=empty(m, f)) if case["save"] else dict(h=empty(m, f))
            return [(ctx.gated_ffn, (desc, state["x"], state["gate"], state["up"], out["h"], out.get("g"), out.get("u")))], out
        out = dict(dx=empty(m, d), dgate=empty(f, d), dup=empty(f, d))
        return [(ctx.gated_ffn_backward, (desc, state["x"], state["gate"], state["up"], state["g"], state["u"], state["dh"], out["dx"],
                                          out["dgate"], out["dup"]))], out
    if op == "matvec":
        desc, out = ctx.int4_desc(dtype, case["group"], case["n"], case["k"]), dict(y=empty(case["rows"], case["n"]))
        return [(ctx.matvec_int4, (desc, case["rows"], state["x"], case["k"] + case["gap"], state["w"], out["y"], case["n"]))], out
    if op == "ffn_int4":
        desc, out = ctx.int4_desc(dtype, case["group"], case["f"], case["d"]), dict(h=empty(case["rows"], case["f"]))
        return [(ctx.gated_ffn_int4, (desc, act, case["rows"], state["x"], case["d"] + case["gap"], state["gate"], state["up"], out["h"],
                                      case["f"]))], out
    desc, out = ctx.int4_desc(dtype, case["group"], case["n"], case["k"]), dict(w=empty(case["n"], case["k"]))
    packed = torch.empty(ctx.int4_packed_bytes(desc), dtype=torch.uint8, device=DEVICE)
    return [(ctx.quantize_int4, (desc, state["w"], case["k"], packed)), (ctx.dequantize_int4, (desc, packed, out["w"], case["k"]))], out


def run(state):
    if not own:
        return _plain(state)
    if "calls" not in state:
        state["calls"], state["out"] = _calls(state)
    for fn, args in state["calls"]:
        fn(*args)
    return state["out"]


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------

def _weights64(packed, n, k, group, dtype):
    """The weights one by one from the places that the layout gives them."""
    across = -(-k // 128)
    col = torch.arange(k, device=DEVICE)
    e = col % 8
    at_col = col // 128 * 1024 + col % 32 // 8 * 256 + col % 128 // 32 * 4 + e % 2 * 2 + e // 4    # byte of the tile row that holds it
    shift = 4 * (e // 2 % 2)
    scales = packed[-(-n // 16) * across * 1024:].view(dtype)
    per = 128 // group
    scale_at = col // 128 * 16 * per + col % 128 // group
    w = torch.empty((n, k), dtype=torch.float64, device=DEVICE)
    step = max(16, (1 << 24) // k // 16 * 16)
    for r0 in range(0, n, step):
        r = torch.arange(r0, min(n, r0 + step), device=DEVICE).unsqueeze(1)
        nibble = packed[r // 16 * (across * 1024) + r % 16 * 16 + at_col].to(torch.int64) >> shift & 15
        w[r0: r0 + step] = (nibble - 8) * scales[r // 16 * (across * 16 * per) + r % 16 * per + scale_at].double()
    return w


def _logistic(z):
    return torch.special.expit(z)


def _both64(name, g):
    """act(g) and its derivative"""
    if name == "silu":
        p = _logistic(g)
        return g * p, p + g * p * _logistic(-g)
    if name == "sigmoid":
        return _logistic(g), _logistic(g) * _logistic(-g)
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-g / 2 ** 0.5)
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / (2 * math.pi) ** 0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5    # (1 + tanh z) / 2 is the logistic function at 2 z
        z2, slope = 2 * c * (g + 0.044715 * g ** 3), 2 * c * (1 + 0.134145 * g ** 2)
        p = _logistic(z2)
        return g * p, p + g * p * _logistic(-z2) * slope
    on = g > 0
    return torch.where(on, g, 0.0), on.double()


def exact(case, seed):
    s, op, t = prepare(case, seed), case["op"], TYPES[case["type"]]
    if op == "ffn":
        g, u = (torch.mm(s["x"].double(), s[w].double().t()) for w in ("gate", "up"))
        h = _both64(case["act"], g)[0] * u
        return dict(h=h, g=g, u=u) if case["save"] else dict(h=h)
    if op == "ffn_backward":
        value, slope = _both64(case["act"], s["g"].double())
        du = s["dh"].double() * value
        dg = s["dh"].double() * s["u"].double() * slope
        x, gate, up = (s[n].double() for n in ("x", "gate", "up"))
        return dict(dx=torch.mm(dg, gate) + torch.mm(du, up), dgate=torch.mm(dg.t(), x), dup=torch.mm(du.t(), x))
    if op == "matvec":
        return dict(y=torch.mm(s["x"].double(), _weights64(s["w"], case["n"], case["k"], case["group"], t).t()))
    if op == "ffn_int4":
        g, u = (torch.mm(s["x"].double(), _weights64(s[w], case["f"], case["d"], case["group"], t).t()) for w in ("gate", "up"))
        return dict(h=_both64(case["act"], g)[0] * u)
    w, group = s["w"].double(), case["group"]
    out = torch.empty_like(w)
    for k0 in range(0, case["k"], group):
        part = w[:, k0: k0 + group]
        scale = (part.abs().max(1, keepdim=True).values / 7).to(t).double()
        out[:, k0: k0 + group] = torch.where(scale > 0, (part / scale).round().clamp(-7, 7) * scale, 0.0)
    return dict(w=out)
