"""Op-level drivers over the C ABI (b200_op_*): torch is used only to own device memory and the
stream; every call goes straight into the hand-written CUDA kernels.  There is no fallback: without
the library or a GPU these raise."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from ._lib import B200Error, ConstrainArgs, StepMapsArgs, TreeAcceptArgs, TreeAttnArgs, check, lib


def _p(t):
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _chk(t, dtype=torch.bfloat16):
    assert t.is_cuda and t.is_contiguous() and t.dtype == dtype, (t.device, t.dtype, t.is_contiguous())


def gemm(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """out[t, n] = sum_k x[t, k] w[n, k]; bf16 in, fp32 accumulate, bf16 out."""
    _chk(x), _chk(w)
    T, K = x.shape
    N = w.shape[0]
    out = torch.empty(T, N, dtype=torch.bfloat16, device=x.device)
    check(lib().b200_op_gemm(_p(w), _p(x), _p(out), N, T, K, _stream()))
    return out


def linear_rows(x, w, bias=None, act=0, p=(0.0, 0.0, 0.0), dtype=torch.bfloat16, out=None):
    """A few rows of x against w, one pass over the weights (b200_op_linear_rows); x and w may be wider buffers' leading columns."""
    assert x.is_cuda and w.is_cuda and x.dtype == w.dtype == torch.bfloat16 and x.stride(1) == w.stride(1) == 1
    T, K = x.shape
    N = w.shape[0]
    out = torch.empty(T, N if act < 3 else N // 2, dtype=dtype, device=x.device) if out is None else out
    check(lib().b200_op_linear_rows(_p(x), _p(w), _p(out), _p(bias) if bias is not None else None, T, N, K, x.stride(0), w.stride(0), out.stride(0),
                                    int(out.dtype == torch.float32), act, *p, _stream()))
    return out


def gemm_deferred(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """Pair GEMM in deferred-reduction mode + the generic partial reducer (T <= 512)."""
    _chk(x), _chk(w)
    T, K = x.shape
    N = w.shape[0]
    out = torch.empty(T, N, dtype=torch.bfloat16, device=x.device)
    check(lib().b200_op_gemm_deferred(_p(w), _p(x), _p(out), N, T, K, _stream()))
    return out


PRO_NONE, PRO_NORM = 0, 1
EPI_PLAIN, EPI_RESADD, EPI_SILU, EPI_ROPE_KV, EPI_ARGMAX = 0, 1, 2, 3, 4


def gemm3(x, w, T=None, pro=PRO_NONE, epi=EPI_PLAIN, force=0, ssq_in=None, norm_w=None, eps=1e-5, out=None, ssq_out=None,
          positions=None, slots=None, cos_sin=None, kv_layer=None, q_heads=0, kv_heads=0, argmax_out=None, n_valid=0,
          normed_out=None, norm_w_out=None, pairs=False):
    """The decode-shape fused GEMM (b200_op_gemm3).  x: [rows >= T, K] activations (or the residual for PRO_NORM),
    w: [N, K].  Returns (out, schedule) with schedule = (pairs per tile, stream-K flag, CTAs).  pairs: EPI_SILU or EPI_ROPE_KV
    as one pass over the weights (b200_op_linear_pairs)."""
    from ._lib import Gemm3Args
    _chk(x), _chk(w)
    T = x.shape[0] if T is None else T
    N, K = w.shape
    a = Gemm3Args(N=N, T=T, K=K, x_rows=x.shape[0], pro=pro, epi=epi, force=force, w=w.data_ptr(), x=x.data_ptr(), eps=eps,
                  q_heads=q_heads, kv_heads=kv_heads, n_valid=n_valid)
    if pro == PRO_NORM:
        _chk(norm_w), _chk(ssq_in, torch.float32)
        a.ssq_in, a.ssq_slabs, a.norm_w = ssq_in.data_ptr(), ssq_in.shape[1], norm_w.data_ptr()
    if epi == EPI_PLAIN:
        out = torch.empty(T, N, dtype=torch.bfloat16, device=x.device) if out is None else out
    elif epi == EPI_RESADD:
        _chk(out)                                               # the residual, updated in place
        ssq_out = torch.zeros(T, N // 128, dtype=torch.float32, device=x.device) if ssq_out is None else ssq_out
        a.ssq_out = ssq_out.data_ptr()
        if norm_w_out is not None:                              # fused RMSNorm of the new residual for the next projection
            _chk(norm_w_out)
            normed_out = torch.empty(T, N, dtype=torch.bfloat16, device=x.device) if normed_out is None else normed_out
            a.normed_out, a.norm_w_out = normed_out.data_ptr(), norm_w_out.data_ptr()
    elif epi == EPI_SILU:
        out = torch.empty(T, N // 2, dtype=torch.bfloat16, device=x.device) if out is None else out
    elif epi == EPI_ROPE_KV:
        _chk(out), _chk(positions, torch.int32), _chk(slots, torch.int32), _chk(cos_sin), _chk(kv_layer)
        a.positions, a.slots, a.cos_sin, a.kv_layer = positions.data_ptr(), slots.data_ptr(), cos_sin.data_ptr(), kv_layer.data_ptr()
        a.max_pos = cos_sin.shape[0]
    elif epi == EPI_ARGMAX:
        argmax_out = torch.empty(T, dtype=torch.int32, device=x.device) if argmax_out is None else argmax_out
        a.argmax_out = argmax_out.data_ptr()
    if out is not None:
        a.out, a.ldo = out.data_ptr(), out.stride(0)
    sch = (C.c_int32 * 3)()
    check(lib().b200_op_linear_pairs(C.byref(a), _stream()) if pairs else lib().b200_op_gemm3(C.byref(a), _stream(), sch))
    res = argmax_out if epi == EPI_ARGMAX else (out, ssq_out, normed_out) if (epi == EPI_RESADD and norm_w_out is not None) \
        else (out, ssq_out) if epi == EPI_RESADD else out
    return res, tuple(sch)


def embed(table, ids):
    _chk(table), _chk(ids, torch.int32)
    out = torch.empty(ids.numel(), table.shape[1], dtype=torch.bfloat16, device=table.device)
    check(lib().b200_op_embed(_p(table), _p(ids), _p(out), ids.numel(), table.shape[1], table.shape[0], _stream()))
    return out


def rmsnorm(x, w, eps, residual=None, row_index=None):
    """Returns normed output; `residual` (if given) is updated in place unless row_index is given."""
    _chk(x), _chk(w)
    rows = row_index.numel() if row_index is not None else x.shape[0]
    out = torch.empty(rows, x.shape[1], dtype=torch.bfloat16, device=x.device)
    check(lib().b200_op_rmsnorm(_p(x), _p(residual), _p(w), _p(out), _p(row_index), rows, x.shape[1], eps, _stream()))
    return out


def rope_kvwrite(qkv, positions, slots, cos_sin, kv_layer, q_heads, kv_heads):
    _chk(qkv), _chk(positions, torch.int32), _chk(slots, torch.int32), _chk(cos_sin), _chk(kv_layer)
    check(lib().b200_op_rope_kvwrite(_p(qkv), _p(positions), _p(slots), _p(cos_sin), _p(kv_layer), qkv.shape[0],
                                     q_heads, kv_heads, cos_sin.shape[0], _stream()))


def silu_mul(gu):
    _chk(gu)
    T, I2 = gu.shape
    out = torch.empty(T, I2 // 2, dtype=torch.bfloat16, device=gu.device)
    check(lib().b200_op_silu_mul(_p(gu), _p(out), T, I2 // 2, _stream()))
    return out


def argmax(logits):
    _chk(logits)
    out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    check(lib().b200_op_argmax(_p(logits), _p(out), logits.shape[0], logits.shape[1], logits.stride(0), _stream()))
    return out


def paged_attn(qkv, kv_layer, block_tables, work, q_heads, kv_heads, decode: bool, out=None, split: int = 0):
    """qkv: [T, (Hq+2Hkv)*128] (q read from it), work: int32 [n, 4] = (q_tok0, q_count, q_pos0, seq).
    split >= 1 (decode only): split-KV form with that many CTAs per (work item, KV head)."""
    _chk(qkv), _chk(kv_layer), _chk(block_tables, torch.int32), _chk(work, torch.int32)
    T = qkv.shape[0]
    if out is None:
        out = torch.zeros(T, q_heads * 128, dtype=torch.bfloat16, device=qkv.device)
    if split:
        assert decode
        check(lib().b200_op_paged_attn_decode_split(_p(qkv), qkv.shape[1], _p(out), out.shape[1], _p(kv_layer), _p(block_tables),
                                                    block_tables.shape[1], _p(work), work.shape[0], q_heads, kv_heads,
                                                    128 ** -0.5, split, _stream()))
        return out
    check(lib().b200_op_paged_attn(_p(qkv), qkv.shape[1], _p(out), out.shape[1], _p(kv_layer), _p(block_tables),
                                   block_tables.shape[1], _p(work), work.shape[0], q_heads, kv_heads,
                                   128 ** -0.5, 1 if decode else 0, _stream()))
    return out


def paged_attn_prefill_tc(qkv, kv_layer, block_tables, work, q_heads, kv_heads, out=None):
    """Tensor-core chunked-prefill attention; work: int32 [n, 4] = (q_tok0, q_count <= 64, q_pos0, seq)."""
    _chk(qkv), _chk(kv_layer), _chk(block_tables, torch.int32), _chk(work, torch.int32)
    T = qkv.shape[0]
    if out is None:
        out = torch.zeros(T, q_heads * 128, dtype=torch.bfloat16, device=qkv.device)
    check(lib().b200_op_paged_attn_prefill_tc(_p(qkv), T, qkv.shape[1], _p(out), out.shape[1], _p(kv_layer), _p(block_tables),
                                              block_tables.shape[1], _p(work), work.shape[0], q_heads, kv_heads, 128 ** -0.5, _stream()))
    return out


def prompt_attn(q, kv, lens, scale, q2=None, k2=None, v2=None, window=0, softcap=0.0, sink=None):
    """Attention of whole prompts of `lens` tokens one behind the other (b200_op_prompt_attn): q [T, heads, 128], kv [T, kv_heads, 256]."""
    for t in (q, kv, q2, k2, v2):
        if t is not None:
            _chk(t)
    if sink is not None:
        _chk(sink, torch.float32)
    T, heads, _ = q.shape
    assert sum(lens) == T and min(lens) > 0 and kv.shape[0] == T
    starts = [sum(lens[:i]) for i in range(len(lens))]
    seqs = torch.tensor([[a, n, 0, 0, 0, 0, 0, 0] for a, n in zip(starts, lens)], dtype=torch.int32).to(q.device)
    out = torch.empty(T, heads, 128, dtype=torch.bfloat16, device=q.device)
    check(lib().b200_op_prompt_attn(_p(q), _p(q2), _p(kv), _p(k2), _p(v2), _p(out), T, heads, kv.shape[1], _p(seqs), len(lens), window, scale, softcap, _p(sink), _stream()))
    return out


# ---- a verification step of drafted tokens (b200_op_step_maps and the three behind it)
def _refused(why):
    return B200Error(-1, why)


def _gpu(t):
    """The GPU that a call runs on: its first tensor's, which has to be the current one."""
    at = t.get_device()
    if at < 0 or at != torch._C._cuda_getDevice():
        raise _refused(f"a tensor on {t.device} where the current GPU's are wanted")
    return at


def _ints(at, *tensors):
    """int32, contiguous and on the call's GPU."""
    for t in tensors:
        if t is not None and not (t.dtype is torch.int32 and t.get_device() == at and t.is_contiguous()):
            raise _refused(f"needs contiguous int32 on cuda:{at}, got {t.dtype} on {t.device}{'' if t.is_contiguous() else ', with strides'}")


def _sized(t, n, what):
    if t is not None and t.numel() != n:
        raise _refused(f"{what}: {t.numel()} values, not {n}")


def _rows(at, t, kinds, what, columns=None, rows=None):
    """Rows that may be a wider buffer's leading columns: how far apart they are."""
    shape, stride = t.shape, t.stride()
    if not (t.dtype in kinds and t.get_device() == at and len(shape) == 2 and (rows is None or shape[0] == rows) and (columns is None or shape[1] >= columns) and
            (not t.numel() or ((shape[1] == 1 or stride[1] == 1) and (shape[0] == 1 or stride[0] >= shape[1])))):
        raise _refused(f"{what}: rows [{'any' if rows is None else rows}, {'any' if columns is None else columns}] of {' or '.join(map(str, kinds))} on cuda:{at}, "
                       f"got {t.dtype} {tuple(shape)}, strides {stride}, on {t.device}")
    return stride[0] if shape[0] > 1 and stride[0] > shape[1] else shape[1]


def _mask_words(masks, T):
    """Words of a row of ancestor masks [T, 1 to 8]; 0 where there are none.  (A tensor without words has no address either, which would stand for no masks.)"""
    if masks is None:
        return 0
    if masks.dim() != 2 or masks.shape[0] != T or not 1 <= masks.shape[1] <= 8:
        raise _refused(f"masks: [{T}, 1 to 8 words], got {tuple(masks.shape)}")
    return masks.shape[1]


def _pieces(like, sizes):
    """New int32 tensors of these sizes, one behind the other.  (Not views to autograd, which integers have no part in: 2.8 us for eight in place of 3.7.)"""
    return like.new_empty(sum(sizes)).unsafe_split_with_sizes(sizes)


def _ptr(t):
    return None if t is None else t.data_ptr()


# sizes go to the library as 32 bits: one that does not fit would lose its upper ones
_WIDE = "a size is negative or passes 32 bits"
_I32, _BF16, _LOGITS = (torch.int32,), (torch.bfloat16,), (torch.bfloat16, torch.float32)


class StepMaps(NamedTuple):
    starts: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    seqs: torch.Tensor
    masks: torch.Tensor | None
    held: torch.Tensor
    cursor: torch.Tensor
    status: torch.Tensor


def step_maps(ctx_lens, new_lens, held, block_tables, free_pages, cursor, rows, parents=None, words=0, inplace=False) -> StepMaps:
    """Slots, positions and, with words > 0, ancestor masks of a step's `rows` rows, from each request's cached tokens and its rows of this step; pages that
    requests lack come from free_pages[cursor:] and are entered in block_tables (b200_op_step_maps).  held and cursor are left as they are and returned
    anew, or updated themselves (inplace).  parents [rows]: the number of each row's parent in its request, -1 for none; without them a chain.  A request that pages or
    lengths do not serve (status 1 or 2) keeps its rows, without slots: the operations behind this one leave it out where they are given `status`."""
    at = _gpu(ctx_lens)
    _ints(at, ctx_lens, new_lens, held, free_pages, cursor, parents)
    S = ctx_lens.numel()
    _sized(new_lens, S, "new_lens"), _sized(held, S, "held"), _sized(cursor, 1, "cursor"), _sized(parents, rows, "parents")
    if rows < 0 or not 0 <= words <= 8:
        raise _refused(f"{rows} rows, masks of {words} words")
    ld = _rows(at, block_tables, _I32, "block tables", rows=S)
    if (S | rows | ld | free_pages.numel()) >> 31:
        raise _refused(_WIDE)
    sizes = [S + 1, rows, rows, rows, S, 0 if inplace else S, 0 if inplace else 1, rows * words]
    starts, positions, slots, seqs, status, held_out, cursor_out, masks = _pieces(ctx_lens, sizes)
    if inplace:
        held_out, cursor_out = held, cursor
    a = StepMapsArgs(S, rows, block_tables.shape[1], ld, free_pages.numel(), words, ctx_lens.data_ptr(), new_lens.data_ptr(), held.data_ptr(), free_pages.data_ptr(),
                     cursor.data_ptr(), _ptr(parents), block_tables.data_ptr(), held_out.data_ptr(), cursor_out.data_ptr(), starts.data_ptr(),
                     positions.data_ptr(), slots.data_ptr(), seqs.data_ptr(), masks.data_ptr(), status.data_ptr())
    check(lib().b200_op_step_maps(C.byref(a), torch._C._cuda_getCurrentRawStream(at)))
    return StepMaps(starts, positions, slots, seqs, masks.view(rows, words) if words else None, held_out, cursor_out, status)


def paged_attn_tree(qkv, kv_layer, block_tables, starts, ctx_lens, masks, q_heads, kv_heads, max_tree, max_ctx=0, scale=128 ** -0.5, out=None, status=None):
    """Attention of a step's rows over the paged cache and those rows of their own request that masks [T, words] names, None: all in front and
    itself (b200_op_paged_attn_tree).  qkv: [T, at least q_heads * 128], q first; kv_layer: [pages, 2, kv_heads, 16, 128] with the step's K and V in it.
    max_tree: the most rows of a request; max_ctx: the most tokens in front of them, if known.  status [S]: step_maps' own, whose requests with 1 or 2 are left out.
    Rows that no request owns, and those of one that is left out, are left as they were in `out` and are zeros in a new one."""
    at = _gpu(qkv)
    ldq = _rows(at, qkv, _BF16, "qkv", columns=q_heads * 128)
    if kv_layer.dtype is not torch.bfloat16 or kv_layer.get_device() != at or not kv_layer.is_contiguous() or kv_layer.shape[1:] != (2, kv_heads, 16, 128):
        raise _refused(f"kv_layer: contiguous bf16 [pages, 2, {kv_heads}, 16, 128] on cuda:{at}, got {kv_layer.dtype} {tuple(kv_layer.shape)} on {kv_layer.device}")
    _ints(at, starts, ctx_lens, masks, status)
    S, T = ctx_lens.numel(), qkv.shape[0]
    _sized(starts, S + 1, "starts"), _sized(status, S, "status")
    words = _mask_words(masks, T)
    ld = _rows(at, block_tables, _I32, "block tables", rows=S)
    if (S | T | ldq | ld | max_tree | max_ctx) >> 31:
        raise _refused(_WIDE)
    fresh = out is None
    if fresh:
        out = qkv.new_empty((T, q_heads * 128))
        ldo = q_heads * 128
    else:
        ldo = _rows(at, out, _BF16, "out", columns=q_heads * 128)
        if out.shape[0] < T:
            raise _refused(f"out has {out.shape[0]} rows, not {T}")
        if ldo >> 31:
            raise _refused(_WIDE)
    a = TreeAttnArgs(S, T, q_heads, kv_heads, ldq, ldo, block_tables.shape[1], ld, words, max_tree, max_ctx, fresh, scale,
                     kv_layer.shape[0], qkv.data_ptr(), out.data_ptr(), kv_layer.data_ptr(), block_tables.data_ptr(), starts.data_ptr(), ctx_lens.data_ptr(), _ptr(masks))
    a.status = _ptr(status)
    a.workspace_bytes = check(lib().b200_op_paged_attn_tree_workspace(C.byref(a)))
    workspace = starts.new_empty((a.workspace_bytes + 3) // 4)
    a.workspace = workspace.data_ptr()
    check(lib().b200_op_paged_attn_tree(C.byref(a), torch._C._cuda_getCurrentRawStream(at)))
    return out


def constrain(logits, starts=None, history=None, hist_starts=None, prompt_lens=None, drafts=None, masks=None, penalties=None, bias=None, allow=None,
              allow_rows=None, out=None, pick=True, status=None):
    """Penalties for repeated tokens, biases and grammar masks on logits [T, V] (bf16 or fp32, rows may be a wider buffer's leading columns) and the greedy
    choice; returns (ids [T] or None, the logits that it was made from or None).  b200_op_constrain has the formulas and the lists' meaning.
    history: the requests' texts in front of this step's rows (not row 0's token, which drafts has); prompt_lens [S]: how many tokens of a text are its prompt, rows that carry a part of
    it among them.  penalties: fp32 [S, 3] = repetition, presence, frequency.  bias: (starts [S + 1], ids, fp32 values).  allow: int32 [masks, at least ceil(V / 32)].
    out: None, a type (torch.float32 or torch.bfloat16) for new logits, or a tensor for them, which may be `logits`.  status [S]: step_maps' own.
    ids of rows that no request owns, or one with status 1 or 2, are -1, logits there are not written."""
    at = _gpu(logits)
    ld = _rows(at, logits, _LOGITS, "logits")
    T, V = logits.shape
    _ints(at, starts, history, hist_starts, prompt_lens, drafts, masks, allow_rows, status)
    S = starts.numel() - 1 if starts is not None else T
    _sized(hist_starts, S + 1, "hist_starts"), _sized(prompt_lens, S, "prompt_lens"), _sized(drafts, T, "drafts"), _sized(allow_rows, T, "allow_rows")
    _sized(status, S, "status")
    words = _mask_words(masks, T)
    if penalties is not None and not (penalties.dtype is torch.float32 and penalties.get_device() == at and penalties.is_contiguous() and penalties.shape == (S, 3)):
        raise _refused(f"penalties: fp32 [{S}, 3] on cuda:{at}, got {penalties.dtype} {tuple(penalties.shape)} on {penalties.device}")
    b_starts, b_ids, b_values, b_len = None, None, None, 0
    if bias is not None:
        b_starts, b_ids, b_values = bias
        b_len = b_ids.numel()
        _ints(at, b_starts, b_ids), _sized(b_starts, S + 1, "bias starts"), _sized(b_values, b_len, "bias values")
        if not (b_values.dtype is torch.float32 and b_values.get_device() == at and b_values.is_contiguous()):
            raise _refused(f"bias values: fp32 on cuda:{at}, got {b_values.dtype} on {b_values.device}")
    allow_ld = _rows(at, allow, _I32, "allow", columns=(V + 31) // 32) if allow is not None else 0
    if allow is not None and not allow.shape[0]:      # no request has a grammar: every row's mask is one that is not there
        if allow_rows is None and T:
            raise _refused(f"allow: no masks for {T} rows")
        allow = allow_rows = None
    out_ld = 0
    if out is not None:
        if isinstance(out, torch.dtype):
            if out not in _LOGITS:
                raise _refused(f"logits are kept as bf16 or fp32, not {out}")
            out = torch.empty(T, V, dtype=out, device=logits.device)
        out_ld = _rows(at, out, _LOGITS, "out", rows=T, columns=V)
    said = history.numel() if history is not None else 0
    masks_there = 0 if allow is None else allow.shape[0]
    if (T | ld | out_ld | said | b_len | allow_ld | masks_there) >> 31:
        raise _refused(_WIDE)
    ids = torch.empty(T, dtype=torch.int32, device=logits.device) if pick else None
    a = ConstrainArgs(S, T, V, ld, logits.dtype is torch.float32, out_ld, out is not None and out.dtype is torch.float32, words,
                      said, b_len, masks_there, allow_ld, logits.data_ptr(), _ptr(out), _ptr(ids),
                      _ptr(starts), _ptr(history), _ptr(hist_starts), _ptr(prompt_lens), _ptr(drafts), _ptr(masks), _ptr(penalties), _ptr(b_starts), _ptr(b_ids),
                      _ptr(b_values), _ptr(allow), _ptr(allow_rows), _ptr(status))
    check(lib().b200_op_constrain(C.byref(a), torch._C._cuda_getCurrentRawStream(at)))
    return ids, out


class TreeAccept(NamedTuple):
    accepted: torch.Tensor
    path: torch.Tensor
    tokens: torch.Tensor
    ctx_lens: torch.Tensor


def tree_accept(ids, drafts, parents, starts, ctx_lens, block_tables, kv, max_path, status=None) -> TreeAccept:
    """The path of drafts that the choices `ids` confirm in each request's tree (parents None: a chain), and its K and V moved to the positions behind the cached
    tokens in every layer of kv [layers, pages, 2, kv_heads, 16, 128], None: nowhere (b200_op_tree_accept).  Returns the paths' lengths, rows and chosen tokens (-1 behind
    the last) and the requests' new lengths.  status [S]: step_maps' own, whose requests with 1 or 2 accept nothing."""
    at = _gpu(ids)
    _ints(at, ids, drafts, parents, starts, ctx_lens, status)
    S, T = ctx_lens.numel(), ids.numel()
    _sized(starts, S + 1, "starts"), _sized(drafts, T, "drafts"), _sized(parents, T, "parents"), _sized(status, S, "status")
    layers, pages, heads, apart = 0, 0, 1, 0
    if kv is not None:
        shape = kv.shape
        if not (kv.dtype is torch.bfloat16 and kv.get_device() == at and len(shape) == 6 and shape[2] == 2 and shape[4:] == (16, 128) and (kv.is_contiguous() or not len(kv) or kv[0].is_contiguous())):
            raise _refused(f"kv: bf16 [layers, pages, 2, kv_heads, 16, 128] on cuda:{at}, got {kv.dtype} {tuple(shape)} on {kv.device}")
        layers, pages, heads = shape[0], shape[1], shape[3]
        apart = kv.stride(0) if layers > 1 else 0
    if not 1 <= max_path <= 256:
        raise _refused(f"paths of {max_path} rows")
    ld = _rows(at, block_tables, _I32, "block tables", rows=S)
    if (S | T | layers | heads | ld) >> 31:
        raise _refused(_WIDE)
    sizes = [S, S, S * max_path, S * max_path]
    accepted, ctx, path, tokens = _pieces(ids, sizes)
    a = TreeAcceptArgs(S, T, block_tables.shape[1], ld, max_path, layers, heads, pages, apart, ids.data_ptr(), drafts.data_ptr(), _ptr(parents),
                       starts.data_ptr(), ctx_lens.data_ptr(), block_tables.data_ptr(), _ptr(kv), accepted.data_ptr(), path.data_ptr(), tokens.data_ptr(), ctx.data_ptr(), _ptr(status))
    check(lib().b200_op_tree_accept(C.byref(a), torch._C._cuda_getCurrentRawStream(at)))
    return TreeAccept(accepted, path.view(S, max_path), tokens.view(S, max_path), ctx)


def init_uniform(n, seed, scale, offset, device="cuda"):
    out = torch.empty(n, dtype=torch.bfloat16, device=device)
    check(lib().b200_op_init_uniform(_p(out), n, seed & 0xFFFFFFFF, scale, offset, _stream()))
    return out
