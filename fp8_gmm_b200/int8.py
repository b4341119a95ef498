"""Experts in 8-bit integers: inference forms of GroupedLinear and GroupedMlp.

Weights are quantised once with a scale per output channel, activations on the fly with a scale per row, so no amax
history is needed: a trained module can be evaluated or served on any batch, from one token up.  Kernels:
fp8_gmm_b200/csrc/int8_quantize.cu, int8_gemm.cu.  The reference has FP8 only.

    experts = Int8GroupedMlp.from_mlp(mlp)                                   # after training, or refresh(mlp) after a step
    weights, selected = routing.topk(router_logits, top_k)
    indices, bin_ids, bins, sizes = routing.indices_and_bins(selected, n_experts)
    rows = experts(tokens, sizes, indices=indices, top_k=top_k)              # sizes stay on the GPU
    out = routing.scatter(rows, indices, bin_ids, weights, bins, top_k)
"""
import torch

from . import backend


def _buffers(module, name, groups, n, k, device):
    module.register_buffer(name, torch.zeros(groups, n, k, dtype=torch.int8, device=device))
    module.register_buffer(name + "_scales", torch.zeros(groups, n, dtype=torch.float32, device=device))


class Int8GroupedLinear(torch.nn.Module):
    """``out[rows of group g] = input[rows of group g] @ weight[g].T`` with int8 operands; no gradient."""

    def __init__(self, in_features, out_features, num_groups, device="cuda"):
        super().__init__()
        self.in_features, self.out_features, self.num_groups = in_features, out_features, num_groups
        _buffers(self, "weight", num_groups, out_features, in_features, device)

    @classmethod
    def from_linear(cls, linear):
        """From a GroupedLinear (its bf16 weights)."""
        g, n, k = linear.weight_tensor.shape
        return cls(k, n, g, linear.weight_tensor.device).refresh(linear)

    @torch.no_grad()
    def refresh(self, linear):
        """Quantises the weights again, into the same memory (graphs captured over this module stay valid)."""
        backend.quantize_rows_int8(linear.weight_tensor, codes=self.weight, scales=self.weight_scales)
        return self

    @torch.no_grad()
    def forward(self, input, group_sizes, indices=None, top_k=1):
        """``group_sizes`` on the host or on the GPU (backend.int8_gmm); with ``indices`` (routing.indices_and_bins)
        ``input`` holds the tokens and the result the rows sorted by expert."""
        return backend.int8_linear(input, self.weight, group_sizes, self.weight_scales, indices, top_k)


class Int8GroupedMlp(torch.nn.Module):
    """Two-layer experts ``fc2(act(fc1(x)))`` with int8 operands, bf16 between the layers; no gradient."""

    def __init__(self, in_features, out_features, num_groups, device="cuda", activation="gelu"):
        super().__init__()
        assert activation in ("gelu", "swiglu")
        self.num_groups, self.activation = num_groups, activation
        _buffers(self, "fc1_weight", num_groups, out_features * (2 if activation == "swiglu" else 1), in_features, device)
        _buffers(self, "fc2_weight", num_groups, in_features, out_features, device)

    @classmethod
    def from_mlp(cls, mlp):
        """From a GroupedMlp (its bf16 weights)."""
        g, hidden, ffn = mlp.fc2_weight.shape
        return cls(hidden, ffn, g, mlp.fc2_weight.device, mlp.activation).refresh(mlp)

    @torch.no_grad()
    def refresh(self, mlp):
        """Quantises the weights again, into the same memory (graphs captured over this module stay valid)."""
        backend.quantize_rows_int8(mlp.fc1_weight, codes=self.fc1_weight, scales=self.fc1_weight_scales)
        backend.quantize_rows_int8(mlp.fc2_weight, codes=self.fc2_weight, scales=self.fc2_weight_scales)
        return self

    @torch.no_grad()
    def forward(self, input, group_sizes, indices=None, top_k=1):
        """Arguments as in Int8GroupedLinear.forward."""
        pre = backend.int8_linear(input, self.fc1_weight, group_sizes, self.fc1_weight_scales, indices, top_k)
        return backend.int8_linear(pre, self.fc2_weight, group_sizes, self.fc2_weight_scales, activation=self.activation)
