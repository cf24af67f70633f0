"""The next token of a batch from the caller's uniform numbers, on torch tensors.

sample() applies temperature, top-k, top-p and min-p per row and draws one
token per row on the device (hc_sample_uniform_dev).  hypno's own sampler with
its XorShift64 states is engine.DeviceSampler.
"""
import torch

from . import _lib
from ._lib import check, load, raw_stream

__all__ = ["sample"]


def _per_row(x, name, dtype, rows, device):
    if not isinstance(x, torch.Tensor):
        return torch.full((rows,), x, dtype=dtype, device=device)
    if x.dtype is not dtype or x.dim() != 1 or x.shape[0] != rows or x.get_device() != device.index:
        raise TypeError(f"{name} must be a number or a [{rows}] {dtype} tensor on {device}")
    if x.stride(0) != 1 and rows > 1:
        raise ValueError(f"{name} must be contiguous")
    return x


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, logprob=None):
    """Draws one token for each row of logits ([rows, vocab] float32, any row
    stride) from u ([rows] float32 in [0, 1)).  temperature, top_p, min_p
    (float32) and top_k (int32) are numbers or [rows] tensors.

    Tokens are ordered by logit, equal ones by index.  Kept are the first top_k
    (0: all), of these every token with less than top_p of their probability
    before it (1: all), of these the ones with at least min_p times the largest
    probability (0: all), and always the first.  temperature 0 keeps the first
    alone.  The token is the first kept index whose running mass exceeds u
    times the kept mass.  Returns (tokens int32 [rows], the log of each token's
    share of the kept mass); -1 and -inf for a row without a logit above -inf."""
    if not isinstance(logits, torch.Tensor) or logits.dtype != torch.float32 or logits.dim() != 2 or not logits.is_cuda:
        raise TypeError("logits must be a 2-dimensional float32 CUDA tensor")
    rows, vocab = logits.shape
    dev = logits.device
    if _lib.current_device() != dev.index:
        with _lib.on_device(dev.index):
            return sample(logits, u, temperature, top_k, top_p, min_p, out, logprob)
    if vocab < 1:
        raise ValueError("logits without a vocabulary")
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("the rows of logits must be contiguous")
    f, i = torch.float32, torch.int32
    u = _per_row(u, "u", f, rows, dev)
    t = _per_row(temperature, "temperature", f, rows, dev)
    k = _per_row(top_k, "top_k", i, rows, dev)
    p = _per_row(top_p, "top_p", f, rows, dev)
    m = _per_row(min_p, "min_p", f, rows, dev)
    out = torch.empty_like(k) if out is None else _per_row(out, "out", i, rows, dev)
    logprob = torch.empty_like(t) if logprob is None else _per_row(logprob, "logprob", f, rows, dev)
    ld = logits.stride(0) if rows > 1 else vocab
    if ld < vocab:
        raise ValueError("the rows of logits overlap")
    check(load().hc_sample_uniform_dev(logits.data_ptr(), ld, rows, vocab, u.data_ptr(), t.data_ptr(), k.data_ptr(),
                                       p.data_ptr(), m.data_ptr(), out.data_ptr(), logprob.data_ptr(),
                                       raw_stream(dev.index)))
    return out, logprob
