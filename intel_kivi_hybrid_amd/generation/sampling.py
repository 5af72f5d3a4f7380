"""Next-token selection for the ``generate()`` loop
(src/kivi_sycl/generation/sampling.py:10-25 in the reference)."""

from typing import Optional

import torch

__all__ = ["sample_token"]


def sample_token(logits: torch.Tensor, temperature: float, top_k: Optional[int],
                 do_sample: bool, top_p: Optional[float] = None,
                 min_p: Optional[float] = None) -> torch.Tensor:
    """``logits [B, V]`` -> next ids ``[B, 1]``.

    Greedy (``do_sample=False``) is the argmax.  Sampling divides by
    ``max(temperature, 1e-8)``, masks everything below the k-th largest logit
    to -inf when ``top_k`` is set, and draws from the softmax.

    With ``top_p`` or ``min_p`` the draw is :func:`_C.sample`'s, on the GPU (where
    logits from the host are copied to), with a random number for each row from
    torch's generator of the logits' device: exactly ``top_k`` tokens, of these the
    most likely with ``top_p`` of the mass, of these the ones at least ``min_p``
    times as likely as the first."""
    if not do_sample:
        return logits.argmax(dim=-1).unsqueeze(1)
    if top_p is not None or min_p is not None:
        return _sample_cut(logits, max(temperature, 1e-8), top_k, top_p, min_p)
    scaled = logits / max(temperature, 1e-8)
    if top_k is not None:
        kth = scaled.topk(top_k, dim=-1).values[:, -1:]
        scaled = scaled.masked_fill(scaled < kth, float("-inf"))
    return torch.multinomial(torch.softmax(scaled, dim=-1), num_samples=1)


def _sample_cut(logits, temperature, top_k, top_p, min_p):
    from .. import _C
    u = torch.rand(logits.shape[0], dtype=torch.float64, device=logits.device)
    at = logits.device if logits.is_cuda else torch.device("cuda")
    ids = _C.sample(logits.to(at), u.to(at), temperature=temperature,
                    top_k=0 if top_k is None else top_k,
                    top_p=1.0 if top_p is None else top_p,
                    min_p=0.0 if min_p is None else min_p).to(logits.device)
    if bool((ids < 0).any()):                # (the caller's next step would read row -1)
        raise ValueError("a row of logits has none above -infinity")
    return ids.unsqueeze(1)
