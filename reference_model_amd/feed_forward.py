"""The feed-forward operators together, as a program uses them: a gated block is trained in bf16, its weights are quantised to 4 bits, and single
tokens are answered from those.

    python -m reference_model_amd.feed_forward [--rows 512] [--width 512] [--hidden 1408] [--steps 60] [--group 32] [--tokens 64]

The block learns another one's answers (random weights, random inputs).  Prints the loss on the way, what the 4-bit weights are off by, how far the
answers from them are from those of the 16-bit block, and the time of a token through one captured graph.
"""
import argparse

from . import capi
from .capi import Context


def train(ctx, desc, x, target, gate, up, steps, rate):
    """Gradient descent on sum((h - target)^2) / 2 per row; gate and up (bf16) follow weights in 32 bits.  Returns the mean loss of every step."""
    import torch

    rows, hidden = target.shape
    h, pre_gate, pre_up = (torch.empty(rows, hidden, device=x.device, dtype=x.dtype) for _ in range(3))
    d_gate, d_up = torch.empty_like(gate), torch.empty_like(up)
    masters, losses = [gate.float(), up.float()], []
    for _ in range(steps):
        ctx.gated_ffn(desc, x, gate, up, h, pre_gate, pre_up)
        off = h.float() - target.float()
        losses.append((off * off).mean())
        ctx.gated_ffn_backward(desc, x, gate, up, pre_gate, pre_up, (off / rows).to(x.dtype), None, d_gate, d_up)
        for master, stored, gradient in zip(masters, (gate, up), (d_gate, d_up)):
            master -= rate * gradient.float()
            stored.copy_(master)
    return [float(v) for v in losses]


class Int4Block:
    """gate, up and down of a block in 4 bits; answers one token or a few"""

    def __init__(self, ctx, activation, group, gate, up, down):
        import torch

        self.ctx, self.activation = ctx, activation
        hidden, width = gate.shape
        dtype = capi.BF16 if gate.dtype == torch.bfloat16 else capi.FP16
        self.into, self.back = ctx.int4_desc(dtype, group, hidden, width), ctx.int4_desc(dtype, group, width, hidden)
        self.gate, self.up, self.down = (self.quantize(desc, w) for desc, w in ((self.into, gate), (self.into, up), (self.back, down)))

    def quantize(self, desc, w):
        import torch

        packed = torch.empty(self.ctx.int4_packed_bytes(desc), device=w.device, dtype=torch.uint8)
        self.ctx.quantize_int4(desc, w, w.stride(0), packed)
        return packed

    def weights(self, desc, packed, like):
        """what the 4-bit weights stand for, in 16 bits"""
        import torch

        w = torch.empty_like(like)
        self.ctx.dequantize_int4(desc, packed, w, w.stride(0))
        return w

    def answer(self, x, h, y):
        """y = down (act(gate x) * (up x)) for the rows of x; h receives the hidden features"""
        self.ctx.gated_ffn_int4(self.into, self.activation, x.shape[0], x, x.stride(0), self.gate, self.up, h, h.stride(0))
        self.ctx.matvec_int4(self.back, x.shape[0], h, h.stride(0), self.down, y, y.stride(0))


def run(rows=512, width=512, hidden=1408, steps=60, group=32, tokens=64, activation=capi.ACT_SILU, rate=0.04):
    """Returns the losses, and relative errors (in the mean of squares) of the 4-bit weights and of the answers from them."""
    import torch

    ctx = Context(0)
    try:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        gen = torch.Generator(device="cuda").manual_seed(1)
        matrix = lambda n, k, std: (torch.randn(n, k, device="cuda", generator=gen) * std).to(torch.bfloat16)  # noqa: E731
        far = lambda a, b: float((a.float() - b.float()).square().mean().sqrt() / b.float().square().mean().sqrt())  # noqa: E731

        x, down = matrix(rows, width, 1.0), matrix(width, hidden, hidden ** -0.5)
        teacher = matrix(hidden, width, width ** -0.5), matrix(hidden, width, width ** -0.5)
        target = torch.empty(rows, hidden, device="cuda", dtype=torch.bfloat16)
        desc = ctx.gated_ffn_desc(capi.BF16, activation, rows, width, hidden)
        ctx.gated_ffn(desc, x, *teacher, target)

        gate, up = (w + matrix(hidden, width, 0.5 * width ** -0.5) for w in teacher)
        losses = train(ctx, desc, x, target, gate, up, steps, rate)

        block = Int4Block(ctx, activation, group, gate, up, down)
        off = far(block.weights(block.into, block.gate, gate), gate)

        # one token after the other; the launches of a token are captured once
        one, h, y = x[:1].clone(), torch.empty(1, hidden, device="cuda", dtype=torch.bfloat16), torch.empty(1, width, device="cuda", dtype=torch.bfloat16)
        block.answer(one, h, y)
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            ctx.set_stream(side.cuda_stream)
            block.answer(one, h, y)
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        answers = torch.empty(tokens, width, device="cuda", dtype=torch.bfloat16)
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for i in range(tokens):
            one.copy_(x[i % rows:i % rows + 1])
            graph.replay()
            answers[i] = y[0]
        end.record()
        torch.cuda.synchronize()

        few = x[torch.arange(tokens, device="cuda") % rows].contiguous()
        hidden16 = torch.empty(tokens, hidden, device="cuda", dtype=torch.bfloat16)
        ctx.gated_ffn(ctx.gated_ffn_desc(capi.BF16, activation, tokens, width, hidden), few, gate, up, hidden16)
        wanted = hidden16.float() @ down.float().T
        if ctx.sync() != capi.VALID:
            raise capi.TmiError(ctx.flags, "a feed-forward operator failed")
        return {"losses": losses, "weights_off": off, "answers_off": far(answers, wanted), "us_per_token": begin.elapsed_time(end) * 1e3 / tokens}
    finally:
        ctx.close()


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("rows", 512), ("width", 512), ("hidden", 1408), ("steps", 60), ("group", 32), ("tokens", 64)):
        parser.add_argument(f"--{name}", type=int, default=value)
    got = run(**vars(parser.parse_args()))
    losses = got["losses"]
    for i in sorted({0, len(losses) // 4, len(losses) // 2, len(losses) - 1}):
        print(f"step {i:3d}  loss {losses[i]:.5f}")
    print(f"4-bit weights off by {got['weights_off']:.3f}, answers from them by {got['answers_off']:.3f}; {got['us_per_token']:.1f} us a token")


if __name__ == "__main__":
    main()
