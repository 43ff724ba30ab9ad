"""The end of a verify step: which drafted tokens stay, and the token that follows them.

``verify_drafts`` is speculative sampling from given random numbers: the acceptance of a verify step
(``demo/src/execution/cb_executor.py:261-300``) in the sampled form of
``pre_exp/moe_spec_acc_rate_benchmark/spec_sampling.py:3-198``, greedy at temperature 0, and on a decode
context the sampling of one token per sequence.  One library call (``odsd_verify_drafts``), no host stop.  ``adjust_logits`` is
what stands in front of it: penalties for repeated tokens, biases and grammar masks on the same rows.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Optional, Union

import torch

from . import _lib
from .ops import _ptr, _raw_device, _rows, _same_device, _stream, _wrote

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


def _float_setting(value, n_seqs: int, what: str, dev: int):
    """(tensor or None, number) of a setting that is one number or one per sequence."""
    if isinstance(value, torch.Tensor):
        _same_device(dev, value)
        if value.dtype != torch.float32 or value.numel() != n_seqs:
            raise ValueError(f"{what} must be a number or float32 [{n_seqs}]")
        return value.contiguous(), 1.0
    return None, float(value)


def _lens_on(t: Optional[torch.Tensor], n_seqs: int, what: str, logits: torch.Tensor) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.numel() != n_seqs:
        raise ValueError(f"{t.numel()} {what} for {n_seqs} sequences")
    if t.get_device() != logits.get_device() or t.dtype != torch.int32:
        t = t.to(device=logits.device, dtype=torch.int32)
    return t.contiguous()


def _half_alike(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices of one shape and dtype, rows dense, share elements without being the same."""
    rows, cols = a.shape
    if a.numel() == 0 or a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr():
        return False
    (sa, ca), (sb, _) = a.stride(), b.stride()
    off = b.storage_offset() - a.storage_offset()
    if rows == 1:
        sa = sb = cols
    if ca != 1 and cols > 1:                                # (its rows are copied first)
        return False
    if off == 0 and sa == sb or off >= (rows - 1) * sa + cols or -off >= (rows - 1) * sb + cols:
        return False
    return sa != sb or not cols <= off % max(sa, 1) <= sa - cols


def adjust_logits(logits: torch.Tensor, context: Dict, *, tokens: Optional[torch.Tensor] = None,
                  token_lens: Optional[torch.Tensor] = None, prompt_lens: Optional[torch.Tensor] = None,
                  draft_tokens: Optional[torch.Tensor] = None, repetition: Union[float, torch.Tensor] = 1.0,
                  frequency: Union[float, torch.Tensor] = 0.0, presence: Union[float, torch.Tensor] = 0.0,
                  bias_tokens: Optional[torch.Tensor] = None, bias_values: Optional[torch.Tensor] = None,
                  mask: Optional[torch.Tensor] = None, mask_rows: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The rows that ``verify_drafts`` takes (logits [n_rows, vocab] and context as there), after penalties, biases and masks, in the
    dtype of logits; ``out`` may be logits itself.  In this order, in fp32, rounded once:

    ``repetition`` (> 0): logits of tokens that occurred are divided by it where positive, multiplied where not.  ``frequency``,
    ``presence``: frequency * n + presence [n > 0] is subtracted, n the times that the token was put out.  Each one number or
    float32 [n_seqs].  ``tokens`` int32 / int64 [n_seqs, max_tokens]: what each sequence has so far, ``token_lens`` of them (None: all), the first
    ``prompt_lens`` (None: none) its prompt, which counts for repetition only; row j of a sequence has put out its first j
    ``draft_tokens`` too.  ``bias_tokens`` int32 / ``bias_values`` float32 [n_seqs, m]: added to these tokens' logits (-1: none; of a token
    named twice the later; hundreds of them: for thousands of forbidden tokens take a mask, the time of long lists grows with their
    square).  ``mask`` int32 [n, words of 32]: where bit t % 32 of word t // 32 is clear token t gets -inf; row i has mask
    ``mask_rows[i]`` (None: i; -1: no mask).  Rows of logits behind the last sequence's are left out: out has there what it had."""
    dev = logits.get_device()
    _same_device(dev, tokens, draft_tokens, bias_tokens, bias_values, mask, mask_rows, out)
    if dev != _raw_device():
        with torch.cuda.device(dev):
            return adjust_logits(logits, context, tokens=tokens, token_lens=token_lens, prompt_lens=prompt_lens,
                                 draft_tokens=draft_tokens, repetition=repetition, frequency=frequency, presence=presence,
                                 bias_tokens=bias_tokens, bias_values=bias_values, mask=mask, mask_rows=mask_rows, out=out)
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"logits are float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [n_rows, vocab], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    lens = context.get("verify_query_lens")
    n_seqs = rows if lens is None else lens.numel()
    n_drafts = 0 if draft_tokens is None else draft_tokens.numel()
    if lens is None and n_drafts:
        raise ValueError("drafted tokens need a context with verify_query_lens")
    if lens is not None and not lens.is_cuda and n_seqs:       # readable without a device synchronisation
        host = lens.tolist()
        if min(host) < 0 or sum(host) > rows or (draft_tokens is not None and sum(max(n - 1, 0) for n in host) != n_drafts):
            raise ValueError(f"query lengths {host} do not fit {rows} rows and {n_drafts} drafts")
    lens = _lens_on(lens, n_seqs, "query lengths", logits)
    if draft_tokens is not None:
        draft_tokens = draft_tokens.to(torch.int64).contiguous()
    tp, token_bytes, token_stride, max_tokens = None, 8, 0, 0
    if tokens is not None:
        token_bytes = {torch.int64: 8, torch.int32: 4}.get(tokens.dtype)
        if token_bytes is None:
            raise TypeError("tokens must be int32 or int64")
        if tokens.dim() != 2 or tokens.shape[0] != n_seqs:
            raise ValueError(f"tokens {tuple(tokens.shape)} for {n_seqs} sequences")
        max_tokens = tokens.shape[1]
        tokens, token_stride = _rows(tokens, n_seqs, max_tokens)
        tp = tokens.data_ptr()
        token_lens = _lens_on(token_lens, n_seqs, "token_lens", logits)
        prompt_lens = _lens_on(prompt_lens, n_seqs, "prompt_lens", logits)
    elif token_lens is not None or prompt_lens is not None:
        raise ValueError("lengths without tokens")
    r_t, r = _float_setting(repetition, n_seqs, "repetition", dev)
    f_t, f = _float_setting(frequency, n_seqs, "frequency", dev)
    p_t, p = _float_setting(presence, n_seqs, "presence", dev)
    if not 0.0 < r < float("inf") or not abs(f) < float("inf") or not abs(p) < float("inf"):
        raise ValueError(f"repetition {repetition} must be positive, frequency {frequency} and presence {presence} finite")
    n_bias = 0
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values belong together")
    if bias_tokens is not None:
        if bias_tokens.dim() != 2 or bias_tokens.shape[0] != n_seqs or bias_values.shape != bias_tokens.shape:
            raise ValueError(f"biases must be [{n_seqs}, m]")
        if bias_tokens.dtype != torch.int32 or bias_values.dtype != torch.float32:
            raise TypeError("bias_tokens are int32, bias_values float32")
        n_bias = bias_tokens.shape[1]
        bias_tokens, bias_values = bias_tokens.contiguous(), bias_values.contiguous()
    mp, mask_stride, n_mask = None, 0, 0
    if mask is not None:
        words = (vocab + 31) // 32
        if mask.dtype != torch.int32 or mask.dim() != 2 or mask.shape[1] < words:
            raise ValueError(f"mask must be int32 [n, {words}]")
        n_mask = mask.shape[0]
        if mask_rows is None:
            if n_mask != rows:
                raise ValueError(f"{n_mask} masks for {rows} rows")
        else:
            if mask_rows.dtype != torch.int32 or mask_rows.numel() != rows:
                raise ValueError(f"mask_rows must be int32 [{rows}]")
            mask_rows = mask_rows.contiguous()
        mask, mask_stride = _rows(mask, n_mask, mask.shape[1])
        mp = mask.data_ptr()
    elif mask_rows is not None:
        raise ValueError("mask_rows without masks")
    if (rows | vocab | n_seqs | n_drafts | max_tokens | n_bias | n_mask) >> 31:      # (sizes are 31 bits in the library)
        raise _lib.OdsdError(f"adjust_logits: unsupported sizes: {rows} rows of {vocab}, {max_tokens} tokens, {n_bias} biases, {n_mask} masks")
    given = out is not None
    if given:
        if out.shape != logits.shape or out.dtype != logits.dtype:
            raise ValueError("out must have the shape and dtype of logits")
        if out.numel() and (out.stride(1) != 1 and vocab > 1 or out.stride(0) < vocab and rows > 1):
            raise ValueError("the rows of out must be dense")
        if _half_alike(logits, out):
            raise ValueError("out must be logits itself, or share no element with it")
    else:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    if rows == 0 or vocab == 0 or n_seqs == 0:
        return out
    ldo = out.stride(0) if rows > 1 else vocab
    logits, ld = _rows(logits, rows, vocab)
    rc = _lib.load().odsd_adjust_logits(logits.data_ptr(), ld, out.data_ptr(), ldo, code, rows, vocab, _ptr(lens), n_seqs, tp, token_bytes,
                                        token_stride, max_tokens, _ptr(token_lens), _ptr(prompt_lens), _ptr(draft_tokens), n_drafts,
                                        _ptr(r_t), r, _ptr(f_t), f, _ptr(p_t), p, _ptr(bias_tokens), _ptr(bias_values), n_bias, mp,
                                        mask_stride, n_mask, _ptr(mask_rows), _stream())
    if rc:
        _lib.check(rc, "odsd_adjust_logits")
    if given:
        _wrote(out)
    return out
