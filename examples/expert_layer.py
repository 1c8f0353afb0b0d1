"""A layer of experts with quantized weights, from a token's hidden state to the next one: the router's logits (``matmul``), the choice and the
order of the work (``routing``), the chosen experts' gated products and the way back (``experts``, twice), and the weighted sum onto
the hidden state (``routing.combine``).  Five launches or a few more, and nothing that waits for the host, so that a decode step can be
captured:

    python examples/expert_layer.py [tokens ...]
"""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from cubek_amd import (Activation, ComputeClient, ElemType, Epilogue, QuantLevel, QuantScheme, QuantValue, TensorHandleRef, experts, matmul, quantize,
                       routing)

BF16, F32 = ElemType.BF16, ElemType.F32
ref = TensorHandleRef.from_torch


class Weight:
    """Floats [..., rows, cols], quantized in blocks of 32."""

    def __init__(self, floats: torch.Tensor, value: QuantValue = QuantValue.Q4S):
        self.scheme = QuantScheme.default().with_value(value).with_level(QuantLevel.block([32]))
        flat = floats.reshape(-1, floats.shape[-1]).contiguous()
        codes = torch.empty(self.scheme.packed_shape(flat.shape), dtype=torch.int32, device=floats.device)
        scales = torch.empty(self.scheme.scales_shape(flat.shape), dtype=torch.float32, device=floats.device)
        quantize.launch_dynamic(ComputeClient.current(), ref(flat), ref(codes), ref(scales), self.scheme, F32)
        self.codes, self.scales = codes.view(*floats.shape[:-1], -1), scales.view(*floats.shape[:-1], -1)
        self.handles = ref(self.codes), ref(self.scales)


class ExpertLayer:
    """``y = x + sum_j weight[j] * down[e_j](silu(gate[e_j] x) * up[e_j] x)`` over the ``chosen`` experts of each token."""

    def __init__(self, hidden: int, inner: int, num_experts: int, chosen: int, seed: int = 0, device: str = "cuda"):
        gen = torch.Generator(device).manual_seed(seed)

        def floats(*shape):
            return torch.randn(shape, generator=gen, device=device) * shape[-1] ** -0.5
        self.chosen, self.num_experts = chosen, num_experts
        self.router = Weight(floats(num_experts, hidden), QuantValue.Q8S)
        self.gate_up = Weight(floats(num_experts, 2 * inner, hidden))  # rows of the gate, then those it gates
        self.down = Weight(floats(num_experts, hidden, inner))
        self.hidden, self.inner, self.device = hidden, inner, device

    def buffers(self, tokens: int):
        """What a step of `tokens` tokens writes: allocated once, kept across steps."""
        def empty(*shape, dtype=torch.int32):
            return torch.empty(shape, dtype=dtype, device=self.device)
        pairs = tokens * self.chosen
        b = dict(logits=empty(tokens, self.num_experts, dtype=torch.float32), weights=empty(tokens, self.chosen, dtype=torch.float32),
                 experts=empty(tokens, self.chosen), offsets=empty(self.num_experts + 1), rows=empty(pairs), slots=empty(tokens, self.chosen),
                 inner=empty(pairs, self.inner, dtype=torch.bfloat16), out=empty(pairs, self.hidden, dtype=torch.bfloat16),
                 y=empty(tokens, self.hidden, dtype=torch.bfloat16))
        handles = {name: ref(t) for name, t in b.items()}
        x = ref(b["y"])  # (only its shape counts here)
        size = max(matmul.workspace_bytes(self.router.handles[0], self.router.scheme, x, BF16),
                   routing.workspace_bytes(tokens, self.num_experts, self.chosen),
                   experts.workspace_bytes(self.gate_up.handles[0], self.gate_up.scheme, handles["inner"], BF16, Epilogue(Activation.Silu, gated=True)),
                   experts.workspace_bytes(self.down.handles[0], self.down.scheme, handles["out"], BF16))
        b["workspace"] = empty(max(size, 1), dtype=torch.uint8)
        return b, handles

    def __call__(self, x: torch.Tensor, buffers) -> torch.Tensor:
        client, (b, h) = ComputeClient.current(), buffers
        space = dict(workspace=b["workspace"].data_ptr(), workspace_size=b["workspace"].numel())
        hx = ref(x)
        matmul.launch_ref(client, *self.router.handles, self.router.scheme, hx, h["logits"], BF16, F32, **space)
        routing.launch_ref(client, h["logits"], h["weights"], h["experts"], h["offsets"], h["rows"], h["slots"], F32, **space)
        experts.launch_ref(client, *self.gate_up.handles, self.gate_up.scheme, hx, h["offsets"], h["inner"], BF16, BF16, h["rows"],
                           Epilogue(Activation.Silu, gated=True), **space)
        experts.launch_ref(client, *self.down.handles, self.down.scheme, h["inner"], h["offsets"], h["out"], BF16, BF16, **space)
        routing.combine(client, h["out"], h["slots"], h["weights"], h["y"], BF16, BF16, residual=hx)
        return b["y"]


def main() -> None:
    layer = ExpertLayer(hidden=2048, inner=1408, num_experts=64, chosen=6)
    for tokens in [int(a) for a in sys.argv[1:]] or [1, 16, 1024]:
        x, buffers = torch.randn((tokens, layer.hidden), device="cuda").to(torch.bfloat16), layer.buffers(tokens)
        layer(x, buffers)  # (kernels are loaded before the capture)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer(x, buffers)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        for _ in range(5):
            graph.replay()
        start.record()
        for _ in range(50):
            graph.replay()
        end.record()
        torch.cuda.synchronize()
        print(f"{tokens} tokens: {start.elapsed_time(end) / 50 * 1e3:.1f} us a layer, experts of the first token {buffers[0]['experts'][0].tolist()}")


if __name__ == "__main__":
    main()
