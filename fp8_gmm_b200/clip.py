"""Clipping of gradients by their global norm: the step between backward and the optimizer.

``clip_grad_norm_`` takes the arguments of ``torch.nn.utils.clip_grad_norm_`` in the same places, for the 2-norm, on this
package's kernels (fp8_gmm_b200/csrc/grad_norm.cu).  The reference leaves the step to its caller.
"""
import torch

from . import backend


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None, *, group=None):
    """Scales the gradients of ``parameters`` (one tensor or an iterable) in place so that their global 2-norm is at most
    ``max_norm``; returns the norm before that as a 0-dim float32 CUDA tensor.

    Parameters without a gradient are skipped.  Gradients are dense bfloat16, float16 or float32 tensors on one CUDA device,
    each in memory of its own: one that is listed twice is refused (torch scales it twice).  ``norm_type`` other than 2 and
    a negative ``max_norm`` are refused.  ``foreach`` has no effect: the list is always handled as one.  Nothing waits for
    the GPU unless ``error_if_nonfinite`` asks for a check of the norm (the gradients are then left as they are when it fails).

    ``group``: process group over which ALL of ``parameters`` are sharded, as the experts of an ``ExpertParallelMlp`` are: the
    squares are summed over its ranks, so all of them clip by the same norm.  A parameter that every rank holds (a router)
    would count once per rank: take ``backend.multi_sum_squares`` of both kinds apart, sum that of the shards over the ranks, and
    clip all by ``backend.multi_clip``.  Every rank of the group makes the call, also one without gradients."""
    if float(norm_type) != 2.0:
        raise RuntimeError(f"clip_grad_norm_: norm_type must be 2, not {norm_type!r}")
    if torch.is_tensor(parameters):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not error_if_nonfinite and group is None:
        return backend.multi_clip_grad_norm(grads, max_norm)
    squares = backend.multi_sum_squares(grads)
    if group is not None:
        torch.distributed.all_reduce(squares, op=torch.distributed.ReduceOp.SUM, group=group)
    if error_if_nonfinite and not bool(torch.isfinite(squares.sqrt().float())):   # the norm that would be returned
        raise RuntimeError(f"clip_grad_norm_: the global norm is {float(squares.sqrt())}; the gradients are left as they are")
    return backend.multi_clip(grads, squares, max_norm)
