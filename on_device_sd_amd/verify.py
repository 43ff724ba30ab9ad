"""The end of a verify step: which drafted tokens stay, and the token that follows them.

``verify_drafts`` is speculative sampling from given random numbers: the acceptance of a verify step
(``demo/src/execution/cb_executor.py:261-300``) in the sampled form of
``pre_exp/moe_spec_acc_rate_benchmark/spec_sampling.py:3-198``, greedy at temperature 0, and on a decode
context the sampling of one token per sequence.  One library call (``odsd_verify_drafts``), no host stop.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Optional, Union

import torch

from . import _lib
from .ops import _ptr, _raw_device, _rows, _same_device, _stream

_DTYPES = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


@dataclass
class VerifyResult:
    tokens: torch.Tensor        # int64 [n_seqs, max_query_len]: the kept drafts, the drawn token, -1 behind it
    num_accepted: torch.Tensor  # int32 [n_seqs]: kept drafts of each sequence
    accept_probs: torch.Tensor  # float32 [n_drafts]: min(1, p / q) of every draft, kept or not


def verify_drafts(logits: torch.Tensor, draft_tokens: Optional[torch.Tensor], context: Dict,
                  accept_u: Optional[torch.Tensor], sample_u: torch.Tensor, *,
                  draft_logits: Optional[torch.Tensor] = None,
                  temperature: Union[float, torch.Tensor] = 1.0) -> VerifyResult:
    """logits [n_tokens, vocab] (float32 / bfloat16 / float16): the target's, one row per query token of a verify context
    (``verify_query_lens`` int32 [n_seqs], ``max_query_len``), each sequence's rows one after the other: one per drafted
    token and one behind the last.  ``draft_tokens`` [n_drafts]: those tokens, sequence after sequence; ``draft_logits``
    [n_drafts, vocab] in the dtype of logits: what they were drawn from (None: each was certain, an n-gram table's or a
    greedy draft).  ``accept_u`` float32 [n_drafts], ``sample_u`` float32 [n_seqs]: random numbers in [0, 1).
    ``temperature``: one number or float32 [n_seqs], 0 (in a tensor also what is below, or NaN) for greedy; it divides both
    models' logits.

    Draft j of a sequence is kept while accept_u_j < min(1, p_j / q_j) of its token; then one token is drawn, from
    max(p - q, 0) at the first draft that is not kept, or from p behind the last: the lowest token whose cumulative weight
    exceeds sample_u times the total.  What a token is drawn from is summed in fp64; whether a draft is kept, and accept_probs,
    come from fp32 statistics, good to 2.4e-6 of p / q.  -inf masks a token (a filter for the likeliest tokens is applied to
    the logits before).  Without drafts (``draft_tokens`` and ``accept_u`` None; a decode context) one token per row is
    drawn; lengths of 0 and 1, where the context has them, say which sequences of a padded batch have a row (the others get -1).
    ``max_query_len`` is read from the context; without it tokens has as many columns as there are rows."""
    dev = logits.get_device()
    lens = context.get("verify_query_lens")
    t_tensor = temperature if isinstance(temperature, torch.Tensor) else None
    _same_device(dev, draft_tokens, accept_u, sample_u, draft_logits, t_tensor)
    if dev != _raw_device():
        with torch.cuda.device(dev):
            return verify_drafts(logits, draft_tokens, context, accept_u, sample_u, draft_logits=draft_logits,
                                 temperature=temperature)
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"verification takes float32, bfloat16 or float16 logits, got {logits.dtype}")
    rows, vocab = logits.shape
    n_seqs = sample_u.numel()
    n_drafts = 0 if draft_tokens is None else draft_tokens.numel()
    if (draft_tokens is None) != (accept_u is None) or (accept_u is not None and accept_u.numel() != n_drafts):
        raise ValueError("every drafted token needs its random number in accept_u")
    if sample_u.dtype != torch.float32 or (accept_u is not None and accept_u.dtype != torch.float32):
        raise TypeError("random numbers must be float32")
    if lens is None:
        if n_drafts:
            raise ValueError("drafted tokens need a context with verify_query_lens")
        if rows != n_seqs:
            raise ValueError(f"{rows} rows of logits for {n_seqs} sequences")
        longest = 1
    else:
        if lens.numel() != n_seqs:
            raise ValueError(f"{lens.numel()} query lengths for {n_seqs} random numbers")
        if rows < n_drafts:
            raise ValueError(f"{n_drafts} drafts for {rows} rows of logits")
        if not lens.is_cuda and n_seqs:                     # readable without a device synchronisation
            host = lens.tolist()
            if min(host) < 0 or sum(host) != rows or sum(max(n - 1, 0) for n in host) != n_drafts:
                raise ValueError(f"query lengths {host} do not fit {rows} rows and {n_drafts} drafts")
            if context.get("max_query_len", rows) < max(host):
                raise ValueError("max_query_len is below the longest query")
        if lens.get_device() != dev or lens.dtype != torch.int32:
            lens = lens.to(device=logits.device, dtype=torch.int32)
        lens = lens.contiguous()
        longest = context.get("max_query_len", rows)
    if (n_seqs | longest | rows | n_drafts | vocab) >> 31:     # (sizes are 31 bits in the library)
        raise _lib.OdsdError(f"verify_drafts: unsupported sizes: {n_seqs} sequences of up to {longest} rows, {n_drafts} drafts, "
                             f"{rows} rows of {vocab}")
    ld_draft = vocab
    if draft_logits is not None:
        if draft_logits.shape != (n_drafts, vocab) or draft_logits.dtype != logits.dtype:
            raise ValueError(f"draft_logits must be [{n_drafts}, {vocab}] in the dtype of logits")
        draft_logits, ld_draft = _rows(draft_logits, n_drafts, vocab) if n_drafts else (None, vocab)
    if t_tensor is not None:
        if t_tensor.dtype != torch.float32 or t_tensor.numel() != n_seqs:
            raise ValueError(f"temperature must be a number or float32 [{n_seqs}]")
        t_tensor = t_tensor.contiguous()
        t_all = 0.0
    else:
        t_all = float(temperature)
        if not t_all >= 0.0:
            raise ValueError(f"temperature {temperature} is negative or no number")
    logits, ld = _rows(logits, rows, vocab)
    if draft_tokens is not None:
        if draft_tokens.dtype != torch.int64:
            draft_tokens = draft_tokens.to(torch.int64)
        draft_tokens = draft_tokens.contiguous()
        accept_u = accept_u.contiguous()
    sample_u = sample_u.contiguous()
    device = logits.device
    out = VerifyResult(torch.empty((n_seqs, longest), dtype=torch.int64, device=device),
                       torch.empty(n_seqs, dtype=torch.int32, device=device),
                       torch.empty(n_drafts, dtype=torch.float32, device=device))
    if n_seqs == 0 or longest == 0:
        out.num_accepted.zero_()
        out.accept_probs.zero_()
        return out
    lib = _lib.load()
    nbytes = lib.odsd_verify_workspace_bytes(n_seqs, longest, rows, n_drafts, vocab, 0 if draft_logits is None else 1)
    if nbytes == 0:
        raise _lib.OdsdError(f"verify_drafts: unsupported sizes: {n_seqs} sequences, {rows} rows of {vocab}")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    rc = lib.odsd_verify_drafts(logits.data_ptr(), ld, _ptr(draft_logits), ld_draft, code, _ptr(draft_tokens), _ptr(lens),
                                _ptr(t_tensor), t_all, _ptr(accept_u), sample_u.data_ptr(), n_seqs, longest, rows,
                                n_drafts, vocab, out.tokens.data_ptr(), out.num_accepted.data_ptr(),
                                out.accept_probs.data_ptr(), ws.data_ptr(), nbytes, _stream())
    if rc:
        _lib.check(rc, "odsd_verify_drafts")
    return out
