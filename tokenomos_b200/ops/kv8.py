"""The 8-bit cache's operators: the quantised write, attention over it, and the copying of cache rows.

A paged state of such a cache is two tensors: ``pool`` [pages, 2, kv_heads, page, head_dim] of ``torch.float8_e4m3fn`` and
``scales`` [pages, 2, kv_heads] float32, one power of two for each block (the positions of a page, keys or values, one KV
head). A byte stands for ``scale * e4m3``; a block's scale is the smallest with which its largest magnitude fits (between
2^-40 and 2^40). A token whose keys or values of a head are not finite, or above 448 * 2^40, is marked: what sees it is NaN.
"""

from __future__ import annotations

import array
import functools
from typing import Sequence

import torch

from tokenomos_b200 import ops
from tokenomos_b200.ops import _lib
from tokenomos_b200.ops._lib import BF16, F32, KernelError

KV8_DTYPE = torch.float8_e4m3fn


def _here(name: str, *tensors: torch.Tensor | None) -> None:
    """Every tensor on the current device, whose stream the launch goes to."""
    found = -1
    for t in tensors:
        if t is not None:
            device = t.get_device()
            if device < 0:
                ops._cuda(t)
            if found < 0:
                found = torch._C._cuda_getDevice()
            if device != found:
                raise KernelError(f"{name}: a tensor on {t.device} while cuda:{found} is the current device")


def _check_cache(name: str, pool: torch.Tensor, scales: torch.Tensor) -> tuple[int, int, int]:
    """(kv_heads, page, head_dim) of an 8-bit cache."""
    shape = pool.shape
    if len(shape) != 5 or pool.dtype != KV8_DTYPE or shape[1] != 2 or not pool.is_contiguous():
        raise KernelError(f"{name}: the cache is a contiguous {KV8_DTYPE} [pages, 2, kv_heads, page, head_dim] tensor, "
                          f"got {pool.dtype} {tuple(shape)}")
    if shape[0] * 2 * shape[2] * shape[3] >= 1 << 31:
        raise KernelError(f"{name}: a cache of {tuple(shape)} has more rows than 31 bits count")
    if scales.dtype != torch.float32 or scales.shape != shape[:3] or not scales.is_contiguous():
        raise KernelError(f"{name}: the scales are a contiguous float32 {tuple(shape[:3])} tensor, got "
                          f"{scales.dtype} {tuple(scales.shape)}")
    return shape[2], shape[3], shape[4]


def _check_layout(name: str, tokens: int, positions: torch.Tensor, tok_seq: torch.Tensor, block_table: torch.Tensor) -> None:
    if ops._i32(positions, "positions").numel() < tokens or ops._i32(tok_seq, "tok_seq").numel() < tokens:
        raise KernelError(f"{name}: positions or tok_seq is shorter than the {tokens} rows")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or (block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise KernelError(f"{name}: block_table is an int32 [sequences, blocks] tensor with contiguous rows")


def kv8_supported(heads: int, kv_heads: int, head_dim: int) -> bool:
    """Whether the 8-bit cache's operators take a layer: heads of 64 or 128, at most 16 query heads a KV head."""
    return bool(_lib.call("tk_attn_kv8_supported", heads, kv_heads, head_dim))


def qk_norm_rope_write8(qkv: torch.Tensor, pool: torch.Tensor | None, scales: torch.Tensor | None, wq: torch.Tensor | None,
                        wk: torch.Tensor | None, eps: float, inv_freq: torch.Tensor, positions: torch.Tensor,
                        tok_seq: torch.Tensor, block_table: torch.Tensor | None, heads: int, kv_heads: int, head_dim: int, page: int,
                        cs_mult: float = 1.0, interleaved: bool = False) -> torch.Tensor:
    """``qk_norm_rope_write`` for an 8-bit cache: norm (``wq``, ``wk``: both or neither) and rotate the q and k heads of
    ``qkv`` [T, (H + 2 Hkv) D] (rows may be strided); returns q [T, H, D] and writes k and v into ``pool`` and ``scales`` at each token's
    position. ``inv_freq`` [R / 2]: the first R columns are rotated, pairs (i, i + R / 2), or (2i, 2i + 1) when
    ``interleaved``; cos and sin are multiplied by ``cs_mult``. Everything is 32-bit (an angle in two 32-bit numbers) and rounded once; a head whose
    squares overflow 32 bits is 0, as in ``qk_norm_rope_write``. ``kv_heads`` 0: queries only (the layer reads another layer's cache).

    A sequence's tokens lie side by side in the step, at consecutive positions (negative ones are not written), and a page that tokens are written into
    belongs to one sequence. A block that already holds tokens of earlier steps keeps its scale or raises it, and then its earlier bytes are
    rounded to the new one (which changes nothing above 2^-6 of it, e4m3's smallest normal number)."""
    name = "qk_norm_rope_write8"
    _here(name, qkv, pool, scales, wq, wk, inv_freq, positions, tok_seq, block_table)
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.shape[1] != (heads + 2 * kv_heads) * head_dim:
        raise KernelError(f"{name}: qkv {tuple(qkv.shape)} for {heads}+2*{kv_heads} heads of {head_dim}")
    code = ops._dtype_code(qkv)
    T = qkv.shape[0]
    if kv_heads:
        if pool is None or scales is None or block_table is None:
            raise KernelError(f"{name}: keys need a cache, its scales and a block table")
        if _check_cache(name, pool, scales) != (kv_heads, page, head_dim):
            raise KernelError(f"{name}: cache {tuple(pool.shape)} does not match [pages, 2, {kv_heads}, {page}, {head_dim}]")
        _check_layout(name, T, positions, tok_seq, block_table)
    else:
        pool = scales = block_table = wk = None
        if ops._i32(positions, "positions").numel() < T:
            raise KernelError(f"{name}: positions is shorter than the {T} rows")
    rot = 2 * inv_freq.numel()
    ops._f32vec(inv_freq, "inv_freq", rot // 2)
    q = qkv.new_empty((T, heads, head_dim))
    _lib.call("tk_qk_norm_rope_write8", qkv.data_ptr(), qkv.stride(0) if T > 1 else qkv.shape[1], q.data_ptr(), ops._ptr(pool),
              ops._ptr(scales), ops._ptr(ops._f32vec(wq, "q_norm weight", head_dim)), ops._ptr(ops._f32vec(wk, "k_norm weight", head_dim)),
              float(eps), inv_freq.data_ptr(), float(cs_mult), int(bool(interleaved)), positions.data_ptr(), tok_seq.data_ptr(),
              ops._ptr(block_table), block_table.stride(0) if kv_heads else 0, T, heads, kv_heads, head_dim, rot, page, code, ops._stream())
    return q


def _check_attention(name, q, pool, scales, out, positions, tok_seq, block_table, gate, *lists):
    _here(name, q, pool, scales, out, positions, tok_seq, block_table, gate, *lists)
    Hkv, P, D = _check_cache(name, pool, scales)
    shape, dtype = q.shape, q.dtype
    if (len(shape) != 3 or shape[2] != D or shape[1] % Hkv or out.shape != shape or out.dtype != dtype
            or not (q.is_contiguous() and out.is_contiguous())):
        raise KernelError(f"{name}: contiguous q and out [T, H, {D}] of one type, H a multiple of {Hkv}; got {tuple(shape)} "
                          f"{dtype} and {tuple(out.shape)} {out.dtype}")
    T, H, _ = shape
    code = ops._dtype_code(q)
    _check_layout(name, T, positions, tok_seq, block_table)
    if gate is not None and (gate.dtype != q.dtype or tuple(gate.shape) != (T, H) or gate.stride(1) != 1):
        raise KernelError(f"{name}: gate must be a {q.dtype} [T, {H}] view with unit column stride")
    return T, H, Hkv, P, D, code


_sm_count: dict = {}


def _sms(device: int) -> int:
    n = _sm_count.get(device)
    if n is None:
        n = _sm_count[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return n


def _attend(q, pool, scales, out, positions, tok_seq, block_table, tok0, ntok, items, nsplit, rows, shape, window, scale, longest, gate, sink):
    """``nsplit`` 0: the entry point chooses; above 1 the shares of a tile of ``rows`` rows meet in scratch memory."""
    T, H, Hkv, P, D, code = shape
    scratch = None
    if nsplit > 1:
        scratch = torch.empty(items * Hkv * nsplit * rows * (D + 4), dtype=torch.float32, device=q.device)
    _lib.call("tk_attn_kv8", q.data_ptr(), pool.data_ptr(), scales.data_ptr(), out.data_ptr(), positions.data_ptr(), tok_seq.data_ptr(),
              block_table.data_ptr(), block_table.stride(0), ops._ptr(tok0), ops._ptr(ntok), items, H, Hkv, D, P, int(window or 0),
              float(scale), nsplit, int(longest), T, ops._ptr(scratch), ops._ptr(gate), gate.stride(0) if gate is not None else 0,
              1 if sink else 0, code, ops._stream())


@functools.lru_cache(maxsize=None)
def _decode_chooses(page: int, code: int) -> bool:
    """Whether the entry point chooses the shares of single tokens itself (the tcgen05 kernel, which needs no scratch memory)."""
    return bool(_lib.call("tk_attn_kv8_single_tc", page, code))


@functools.lru_cache(maxsize=None)
def _prefill_chooses(heads: int, kv_heads: int, head_dim: int, page: int, code: int) -> bool:
    """The same of prompt portions."""
    return bool(_lib.call("tk_attn_kv8_prefill_supported", heads, kv_heads, head_dim, page, code))


def attention_kv8_decode(q: torch.Tensor, pool: torch.Tensor, scales: torch.Tensor, out: torch.Tensor, positions: torch.Tensor,
                         tok_seq: torch.Tensor, block_table: torch.Tensor, tok_index: torch.Tensor | None, window: int | None,
                         scale: float, longest: int, gate: torch.Tensor | None = None, sink: bool = False) -> None:
    """Causal attention of sequences that bring one token (``tok_index``: their rows of ``q`` [T, H, D], negative ones skipped;
    None: every row is one, in order) over an 8-bit cache that holds this step's keys; writes those rows of ``out``. ``window``: as in
    ``attention``. ``longest``: an upper bound of the positions any of the sequences holds, this token's included; it only picks how many ways
    a row's keys are shared out. ``gate`` [T, H]: the per-head output gate, ``round(o) * round(sigmoid(gate))``; ``sink``: the
    softmax's denominator has one term more, a key of score 0 without a value."""
    name = "attention_kv8_decode"
    shape = _check_attention(name, q, pool, scales, out, positions, tok_seq, block_table, gate, tok_index)
    n = shape[0] if tok_index is None else ops._i32(tok_index, "tok_index").numel()
    if n:
        T, H, Hkv, P, D, code = shape
        nsplit = 0
        if not _decode_chooses(P, code):
            nsplit = _lib.call("tk_attn_kv8_splits", n, H, Hkv, D, P, code, int(longest), abs(int(window)) if window else int(longest), 1,
                               _sms(q.get_device()))
        _attend(q, pool, scales, out, positions, tok_seq, block_table, tok_index, None, n, nsplit, H // Hkv, shape, window, scale, longest,
                gate, sink)


def attention_kv8_tokens(heads: int, kv_heads: int, head_dim: int, page: int, dtype: torch.dtype) -> int:
    """The most tokens of one sequence that a tile of ``attention_kv8_prefill`` has."""
    return _lib.call("tk_attn_kv8_tokens", heads, kv_heads, head_dim, page, F32 if dtype == torch.float32 else BF16)


def attention_kv8_prefill(q: torch.Tensor, pool: torch.Tensor, scales: torch.Tensor, out: torch.Tensor, positions: torch.Tensor,
                          tok_seq: torch.Tensor, block_table: torch.Tensor, tile_tok0: torch.Tensor, tile_ntok: torch.Tensor,
                          window: int | None, scale: float, longest: int, gate: torch.Tensor | None = None,
                          sink: bool = False) -> None:
    """The same for prompt portions: tiles of at most ``attention_kv8_tokens`` tokens of one sequence at consecutive positions (``tile_tok0``:
    each one's first row of ``q``; ``tile_ntok``: its tokens, 0 for an unused entry); writes the tiles' rows of ``out``."""
    name = "attention_kv8_prefill"
    T, H, Hkv, P, D, code = shape = _check_attention(name, q, pool, scales, out, positions, tok_seq, block_table, gate, tile_tok0, tile_ntok)
    n = ops._i32(tile_tok0, "tile_tok0").numel()
    if ops._i32(tile_ntok, "tile_ntok").numel() != n:
        raise KernelError(f"{name}: {n} first tokens for {tile_ntok.numel()} tiles")
    if n:
        nsplit = rows = 0
        if not _prefill_chooses(H, Hkv, D, P, code):
            reach = min(int(longest), abs(int(window)) + T) if window else int(longest)
            rows = _lib.call("tk_attn_kv8_tokens", H, Hkv, D, P, code) * (H // Hkv)
            nsplit = _lib.call("tk_attn_kv8_splits", n, H, Hkv, D, P, code, reach, reach, 0, _sms(q.get_device()))
        _attend(q, pool, scales, out, positions, tok_seq, block_table, tile_tok0, tile_ntok, n, nsplit, rows, shape, window, scale, longest,
                gate, sink)


def attention_kv8_status() -> int:
    """0, or where a warp of the 8-bit cache's attention gave up waiting for its keys since the last call."""
    return _lib.call("tk_attn_kv8_status")


def copy_rows(tensors: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """``t[dst[i]] = t[src[i]]`` for every tensor ``t`` (contiguous, of any type) and every i, in one launch: pages of a cache's layers, or
    requests' state rows. ``src`` and ``dst`` are host integers; no row is a destination twice, and none both a source and a
    destination (refused)."""
    _here("copy_rows", *tensors)
    if len(src) != len(dst):
        raise KernelError(f"copy_rows: {len(src)} sources for {len(dst)} destinations")
    base, row, rows = [], [], []
    for t in tensors:
        shape, size = t.shape, t.nbytes
        if not shape or not t.is_contiguous():
            raise KernelError("copy_rows: contiguous tensors whose first dimension counts the rows")
        if size:
            base.append(t.data_ptr())
            row.append(size // shape[0])
            rows.append(shape[0])
    if not base or not len(src):
        return
    try:
        a, b = array.array("i", src), array.array("i", dst)
    except (TypeError, OverflowError) as exc:
        raise KernelError(f"copy_rows: rows are numbered by 32-bit integers ({exc})") from None
    base, row, rows = array.array("Q", base), array.array("q", row), array.array("i", [min(n, 0x7FFFFFFF) for n in rows])
    _lib.call("tk_copy_rows", base.buffer_info()[0], row.buffer_info()[0], rows.buffer_info()[0], len(rows), a.buffer_info()[0],
              b.buffer_info()[0], len(a), ops._stream())
