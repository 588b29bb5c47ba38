"""Greedy verification of a draft tree (vllm/tree_accept.py): the targets' argmax and the tree walk on gfx950.

Every verify row gets the target's token (greedy: the argmax of its logits, first index on ties). The walk then goes
from the root to the lowest-index child whose draft token equals the current node's token, until a node has no such
child; the accepted rows are the path (root first) and the sampled tokens are the path rows' target tokens, the last
of which is the bonus token.

Where the target samples, :func:`sample_tree` takes that walk's place: it accepts children and draws the bonus token so that
every token is distributed as the target's own.

The reference's module also holds ``TreeRejectionSampler``, vLLM's rejection sampler with the chain rule replaced by
the tree walk (engine glue: it applies the engine's sampling parameters and Gumbel sampling, then calls
:func:`accept_tree`). It is not rewritten here: importing ``TreeRejectionSampler`` from this module runs the installed
eagle-harness's own ``vllm/tree_accept.py`` with its ``accept_tree`` and ``accepted_rows_first`` rebound to this
module's, so every walk it runs is the gfx950 kernel's.
"""

from __future__ import annotations

import torch

from eagle_harness import _overlay
from eagle_harness.kernels import _native
from eagle_harness.vllm.verify_layout import TreeStore

# Names of the reference module that are vLLM engine glue, served from the installed package's own module.
_ENGINE_GLUE = ("TreeRejectionSampler",)


def greedy_targets(logits: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``logits.argmax(-1)`` of ``[rows, vocab]`` logits (bf16 / fp16 / fp32, unit column stride) as int64, first index
    on ties; one gfx950 workgroup per row streams the row with 16-byte loads."""
    rows, vocab = logits.shape
    if logits.stride(1) != 1:
        raise _native.NotCovered("logits must have a unit column stride")
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    elif out.dtype != torch.int64 or not out.is_contiguous() or out.numel() < rows or out.device != logits.device:
        raise ValueError(f"greedy_targets: out must be a contiguous int64 tensor of at least {rows} entries on "
                         f"{logits.device}")
    args = _native.ArgmaxArgs(
        logits=logits.data_ptr(), stride_row=logits.stride(0), dtype=_native.dtype_code(logits.dtype), rows=rows,
        vocab=vocab, out=out.data_ptr(),
    )
    _native.launch("eagle4_argmax_rows", args, logits.device)
    return out


def accept_tree(
    target: torch.Tensor,
    drafted: torch.Tensor,
    cu_num_logits: torch.Tensor,
    idx_mapping: torch.Tensor,
    parents: torch.Tensor,
    store: TreeStore,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The walk for every request (vllm/tree_accept.py:86-115): ``(sampled [num_reqs, W], num_sampled [num_reqs])``;
    the path goes to ``store``. Entries of ``sampled`` past ``num_sampled`` are not written."""
    num_reqs = cu_num_logits.shape[0] - 1
    sampled = drafted.new_empty(num_reqs, store.width)
    num_sampled = torch.empty(num_reqs, dtype=torch.int32, device=target.device)
    args = _native.AcceptTreeArgs(
        target=_native.itab(target),
        drafted=_native.itab(drafted),
        cu_num_logits=_native.itab(cu_num_logits),
        idx_mapping=_native.itab(idx_mapping),
        parents=_native.itab(parents),
        sampled=sampled.data_ptr(),
        stride_sampled=sampled.stride(0),
        num_sampled=num_sampled.data_ptr(),
        path=store.path.data_ptr(),
        stride_path=store.path.stride(0),
        path_len=store.path_len.data_ptr(),
        num_reqs=num_reqs,
        width=store.width,
    )
    if sampled.dtype != torch.int64:
        raise _native.NotCovered("drafted tokens must be int64")
    _native.launch("eagle4_accept_tree", args, target.device)
    return sampled, num_sampled


_LOGIT_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def sample_tree(
    logits: torch.Tensor,
    drafted: torch.Tensor,
    cu_num_logits: torch.Tensor,
    idx_mapping: torch.Tensor,
    parents: torch.Tensor,
    store: TreeStore,
    coins: torch.Tensor,
    final_coins: torch.Tensor,
    temperature: torch.Tensor,
    draft_probs: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Verification by sampling, where :func:`greedy_targets` and :func:`accept_tree` take the argmax: the tokens of the
    walk are distributed as the target's own. ``(sampled [num_reqs, W], num_sampled [num_reqs])`` as
    :func:`accept_tree`'s, entries of ``sampled`` past ``num_sampled`` -1; the path goes to ``store``.

    ``logits`` [rows, vocab] (bf16 / fp16 / fp32, unit column stride; -inf for a token that may not be drawn); ``coins``
    [rows] and ``final_coins`` [num_reqs] fp32 uniform numbers in [0, 1), of a drafted row's acceptance and of the
    token that ends a request's walk; ``temperature`` [num_reqs] fp32 (0: greedy). ``draft_probs`` [rows, vocab] (bf16 /
    fp16 / fp32): row ``n`` what the children of row ``n`` were drawn from, each independently; None where the
    children are the draft's choice and not drawn (its most likely tokens).

    A row's children are tried in row order against the residual ``r`` (first ``p = softmax(logits / temperature)``,
    its mass ``Z = 1``): accepted iff ``coin * q(x) * Z < r(x)``; a rejection leaves ``max(r - Z q, 0)``, or without
    ``draft_probs`` (``q(x) = 1``) ``r`` without ``x``. Without an accepted child the walk ends with the first token
    whose running sum of ``r`` exceeds ``final_coin * Z``. A row whose maximum is not finite has all its mass on its
    argmax. Sums and comparisons are in 64 bits.
    """
    if logits.dim() != 2 or (draft_probs is not None and draft_probs.shape != logits.shape):
        raise ValueError("sample_tree: logits must be [rows, vocab], draft_probs of the same shape")
    (rows, vocab), device = logits.shape, logits.device
    path, path_len, width = store.path, store.path_len, store.width
    num_reqs = cu_num_logits.shape[0] - 1
    row_stride, column = logits.stride()
    prob_stride, prob_column = (0, 1) if draft_probs is None else draft_probs.stride()
    if column != 1 or prob_column != 1:
        raise _native.NotCovered("logits and draft_probs must have a unit column stride")
    if width > 64:
        raise _native.NotCovered(f"tree widths above 64 rows ({width})")
    if logits.dtype not in _LOGIT_DTYPES or (draft_probs is not None and draft_probs.dtype not in _LOGIT_DTYPES):
        raise _native.NotCovered("logits and draft_probs must be bf16, fp16 or fp32, got "
                                 f"{logits.dtype}{'' if draft_probs is None else f', {draft_probs.dtype}'}")
    if drafted.shape != (rows,) or idx_mapping.shape[0] < num_reqs or parents.dim() != 2 or parents.shape[1] < width:
        raise ValueError(f"sample_tree: drafted must be [{rows}], idx_mapping [>= {num_reqs}], parents [slots, >= {width}]")
    for name, t, n in (("coins", coins, rows), ("final_coins", final_coins, num_reqs), ("temperature", temperature, num_reqs)):
        if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] < n or not t.is_contiguous():
            raise ValueError(f"sample_tree: {name} must be a contiguous fp32 vector of {n} entries")
    (path_slots, path_width), (path_stride, path_column) = path.shape, path.stride()
    if (path.dtype != torch.int32 or path_len.dtype != torch.int32 or path_column != 1 or path_width < width
            or not path_len.is_contiguous()):
        raise ValueError("sample_tree: the store's path and path_len must be int32, contiguous over a slot's entries")
    for t in (drafted, cu_num_logits, idx_mapping, parents, coins, final_coins, temperature, draft_probs, path, path_len):
        if t is not None and t.device != device:
            raise ValueError(f"sample_tree: every tensor must be on the logits' device, {device}, got {t.device}")
    itab = _native.itab
    sampled = torch.empty((num_reqs, width), dtype=torch.int64, device=device)
    num_sampled = torch.empty(num_reqs, dtype=torch.int32, device=device)
    args = _native.SampleTreeArgs(
        logits.data_ptr(), row_stride, _native.ptr(draft_probs), prob_stride, itab(drafted), itab(cu_num_logits),
        itab(idx_mapping), itab(parents), coins.data_ptr(), final_coins.data_ptr(), temperature.data_ptr(), sampled.data_ptr(),
        width, num_sampled.data_ptr(), path.data_ptr(), path_stride, path_len.data_ptr(), None, 0, rows, num_reqs, width, vocab,
        min(parents.shape[0], path_slots, path_len.shape[0]), _native.dtype_code(logits.dtype),
        0 if draft_probs is None else _native.dtype_code(draft_probs.dtype))
    need = _native.library().eagle4_sample_tree_workspace(args)
    if need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)  # the torch caching allocator's
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need
    _native.launch("eagle4_sample_tree", args, device)
    return sampled, num_sampled


def accepted_rows_first(
    expanded_idx_mapping: torch.Tensor, expanded_local_pos: torch.Tensor, store: TreeStore
) -> torch.Tensor:
    """Row map of the logits after a tree walk (vllm/tree_accept.py:118-126): entry ``r`` names the logits row that
    row ``r`` must hold. vLLM reads sampled token ``k`` of a request from its ``k``-th logits row, so the first
    ``path_len`` rows of each request take its accepted rows in path order; the rows after them stay in place."""
    row = torch.arange(expanded_local_pos.shape[0], device=expanded_local_pos.device)
    slot = expanded_idx_mapping.long()
    pos = expanded_local_pos.long()
    first_row = row - pos  # the request's first logits row
    on_path = pos < store.path_len[slot]
    return torch.where(on_path, first_row + store.path[slot, pos].long(), row)


def __getattr__(name: str):
    if name in _ENGINE_GLUE:
        glue = _overlay.engine_module(__name__, accept_tree=accept_tree, accepted_rows_first=accepted_rows_first)
        return getattr(glue, name)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
