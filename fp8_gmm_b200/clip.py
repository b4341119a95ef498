"""Clipping of gradients by their global norm: the step between backward and the optimizer.

``clip_grad_norm_`` has the contract of ``torch.nn.utils.clip_grad_norm_`` (2-norm) on this package's kernels
(fp8_gmm_b200/csrc/grad_norm.cu).  The reference leaves the step to its caller.
"""
import torch

from . import backend


def clip_grad_norm_(parameters, max_norm, error_if_nonfinite=False, group=None):
    """Scales the gradients of ``parameters`` (one tensor or an iterable) in place so that their global 2-norm is at most
    ``max_norm``; returns the norm before that as a 0-dim float32 CUDA tensor.

    Parameters without a gradient are skipped.  Nothing waits for the GPU unless ``error_if_nonfinite`` asks for a check of
    the norm (the gradients are then left as they are when it fails).  ``group``: process group over which the
    parameters are sharded, as the experts of an ``ExpertParallelMlp`` are: the squares are summed over its ranks, so all
    of them clip by the same norm.  Every rank of the group makes the call, also one without gradients."""
    if torch.is_tensor(parameters):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not error_if_nonfinite and group is None:
        return backend.multi_clip_grad_norm(grads, max_norm)
    squares = backend.multi_sum_squares(grads)
    if group is not None:
        torch.distributed.all_reduce(squares, op=torch.distributed.ReduceOp.SUM, group=group)
    if error_if_nonfinite and not bool(torch.isfinite(squares)):
        raise RuntimeError(f"clip_grad_norm_: the global norm is {float(squares.sqrt())}; the gradients are left as they are")
    return backend.multi_clip(grads, squares, max_norm)
