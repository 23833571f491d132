"""Rotary positions, attention over a paged K/V cache and drafted tokens: the Python side of flash_rotary, flash_append_paged, flash_forward_paged,
flash_tree_mask and flash_keep_paged (include/flash_attn_mi355.h).

A serving loop keeps K and V in pages of a pool, `[pages, H_kv, page_size, d]`, a table that names each sequence's pages, and the
sequences' lengths.  One step takes the new tokens of all sequences, `[tokens, H, d]`, one after the other:

    q = flash_append_paged(k, v, k_cache, v_cache, table, lens, cu, q=q, inv_freq=inv_freq)
    o, lse = flash_forward_paged(q, k_cache, v_cache, table, lens, cu, max_seqlen_q, max_seqlen_k, causal=True)

A step that checks a tree of drafted tokens per sequence has three more arguments and one more call:

    mask, positions = flash_tree_mask(parents, cu, lens, max_seqlen_q)
    q = flash_append_paged(k, v, k_cache, v_cache, table, lens, cu, q=q, inv_freq=inv_freq, positions=positions)
    o, lse = flash_forward_paged(q, k_cache, v_cache, table, lens, cu, max_seqlen_q, max_seqlen_k, tree_mask=mask)
    lens = flash_keep_paged(k_caches, v_caches, table, lens, cu, path, accepted)   # once the answers have said which path stays

Everything that changes from step to step is read on the GPU (lengths, table, positions, masks, paths), so that a captured graph follows it.
"""
import ctypes as C
import math

from . import binding
from .binding import FLASH_OK, FlashError

_INT_MAX = 2 ** 31 - 1


class RotaryParams(C.Structure):
    """struct flash_rotary_params, field for field."""
    _fields_ = [
        ("X", C.c_void_p), ("Y", C.c_void_p), ("dtype", C.c_int),
        ("B", C.c_int), ("H", C.c_int), ("N", C.c_int), ("d", C.c_int), ("rot", C.c_int),
        ("x_batch", C.c_int64), ("x_head", C.c_int64), ("x_row", C.c_int64),
        ("y_batch", C.c_int64), ("y_head", C.c_int64), ("y_row", C.c_int64),
        ("positions", C.c_void_p), ("positions_64", C.c_int), ("positions_batch", C.c_int64),
        ("inv_freq", C.c_void_p), ("factor", C.c_float), ("interleaved", C.c_int), ("inverse", C.c_int),
    ]


class PagedParams(C.Structure):
    """struct flash_paged_params, field for field."""
    _fields_ = [
        ("Q", C.c_void_p), ("O", C.c_void_p), ("K", C.c_void_p), ("V", C.c_void_p), ("K_cache", C.c_void_p), ("V_cache", C.c_void_p),
        ("block_table", C.c_void_p), ("seqlens_k", C.c_void_p), ("cu_seqlens_q", C.c_void_p), ("dtype", C.c_int),
        ("B", C.c_int), ("H", C.c_int), ("H_kv", C.c_int), ("d", C.c_int),
        ("total_q", C.c_int), ("num_pages", C.c_int), ("page_size", C.c_int), ("max_pages", C.c_int),
        ("q_token", C.c_int64), ("q_head", C.c_int64), ("o_token", C.c_int64), ("o_head", C.c_int64),
        ("k_token", C.c_int64), ("k_head", C.c_int64), ("v_token", C.c_int64), ("v_head", C.c_int64),
        ("kc_page", C.c_int64), ("kc_head", C.c_int64), ("kc_row", C.c_int64), ("vc_page", C.c_int64), ("vc_head", C.c_int64), ("vc_row", C.c_int64),
        ("block_table_stride", C.c_int64),
        ("LSE", C.c_void_p), ("O_partial", C.c_void_p), ("LSE_partial", C.c_void_p),
        ("max_seqlen_q", C.c_int), ("max_seqlen_k", C.c_int), ("softmax_scale", C.c_float),
        ("is_causal", C.c_int), ("window_left", C.c_int), ("window_right", C.c_int), ("num_splits", C.c_int),
        ("inv_freq", C.c_void_p), ("rot", C.c_int), ("interleaved", C.c_int), ("factor", C.c_float),
        ("positions", C.c_void_p), ("positions_64", C.c_int),
        ("softcap", C.c_float), ("alibi_slopes", C.c_void_p), ("prefix_lens", C.c_void_p),
        ("tree_mask", C.c_void_p), ("tree_words", C.c_int), ("tree_stride", C.c_int64),
    ]


FLASH_MIN_SOFTCAP, FLASH_MAX_SOFTCAP = 1e-6, 1000.0
FLASH_MAX_SLOPE = 1024.0
FLASH_MAX_TREE_TOKENS = 256


class TreeParams(C.Structure):
    """struct flash_tree_params, field for field."""
    _fields_ = [
        ("parents", C.c_void_p), ("cu_seqlens_q", C.c_void_p), ("seqlens_k", C.c_void_p), ("mask", C.c_void_p), ("positions", C.c_void_p),
        ("B", C.c_int), ("total_q", C.c_int), ("words", C.c_int), ("mask_stride", C.c_int64),
    ]


class KeepParams(C.Structure):
    """struct flash_keep_params, field for field."""
    _fields_ = [
        ("K_cache", C.c_void_p), ("V_cache", C.c_void_p), ("block_table", C.c_void_p), ("seqlens_k", C.c_void_p), ("cu_seqlens_q", C.c_void_p),
        ("path", C.c_void_p), ("accepted", C.c_void_p), ("seqlens_out", C.c_void_p),
        ("B", C.c_int), ("H_kv", C.c_int), ("d", C.c_int), ("layers", C.c_int), ("num_pages", C.c_int), ("page_size", C.c_int), ("max_pages", C.c_int),
        ("max_path", C.c_int),
        ("kc_layer", C.c_int64), ("kc_page", C.c_int64), ("kc_head", C.c_int64), ("kc_row", C.c_int64),
        ("vc_layer", C.c_int64), ("vc_page", C.c_int64), ("vc_head", C.c_int64), ("vc_row", C.c_int64),
        ("block_table_stride", C.c_int64), ("path_stride", C.c_int64),
    ]


_bound = None


def _lib():
    global _bound
    if _bound is None:
        L = binding.lib()
        rp, pp = C.POINTER(RotaryParams), C.POINTER(PagedParams)
        for name, args in (("flash_rotary", [rp, C.c_void_p]), ("flash_append_paged", [pp, C.c_void_p]), ("flash_forward_paged", [pp, C.c_void_p]),
                           ("flash_tree_mask", [C.POINTER(TreeParams), C.c_void_p]), ("flash_keep_paged", [C.POINTER(KeepParams), C.c_void_p]),
                           ("flash_forward_paged_resolve_splits", [pp]),
                           ("flash_forward_paged_workspace_bytes", [pp, C.POINTER(C.c_size_t), C.POINTER(C.c_size_t)])):
            f = getattr(L, name)
            f.restype, f.argtypes = C.c_int, args
        for name, p in (("flash_rotary_params", RotaryParams), ("flash_paged_params", PagedParams), ("flash_tree_params", TreeParams),
                        ("flash_keep_params", KeepParams)):
            size, init = getattr(L, name + "_size"), getattr(L, name + "_init")
            size.restype, init.restype, init.argtypes = C.c_size_t, None, [C.POINTER(p)]
            if size() != C.sizeof(p):
                raise ImportError(f"the library was built with another {name} ({size()} bytes, this binding: {C.sizeof(p)}): rebuild it")
        _bound = L
    return _bound


class _NoFrontEnd:
    """Leaves every call to this file's own path."""

    @staticmethod
    def rotary(*args):
        return NotImplemented

    append = paged = tree_mask = keep = rotary


_native = None


def _front_end():
    """The native front end (csrc/py_binding.cpp), as binding.py has it."""
    global _native
    L, n = _lib(), binding._native or binding._front_end()
    if hasattr(n, "bind_paged"):
        n.bind_paged(*(C.cast(f, C.c_void_p).value for f in (L.flash_rotary, L.flash_append_paged, L.flash_forward_paged,
                                                             L.flash_forward_paged_resolve_splits, L.flash_tree_mask, L.flash_keep_paged)))
        _native = n
    else:
        _native = _NoFrontEnd
    return _native


def _types():
    import torch

    return {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _check(cond, text):
    if not cond:
        raise ValueError(text)


def _int(v):
    """v as a C int; what lies outside is as good as the nearest one."""
    return max(-_INT_MAX, min(int(v), _INT_MAX))


def _same_device(*tensors):
    """The device of all tensors that are given."""
    device = None
    for t in tensors:
        if t is None:
            continue
        _check(t.is_cuda, "tensors must be on the GPU")
        if device is None:
            device = t.device
        _check(t.device == device, "tensors must be on the same device")
    return device


class _on:
    """The given device current and the given stream, or the device's current one, as the one that results are allocated on."""

    def __init__(self, device, stream):
        import torch

        _check(stream is None or stream.device == device, "the stream must be one of the tensors' device")
        self._device, self._given = torch.cuda.device(device), stream
        self._stream = None

    def __enter__(self):
        import torch

        self._device.__enter__()
        s = self._given
        if s is None:
            s = torch.cuda.current_stream()
        else:
            self._stream = torch.cuda.stream(s)
            self._stream.__enter__()
        return C.c_void_p(s.cuda_stream)

    def __exit__(self, *exc):
        if self._stream is not None:
            self._stream.__exit__(*exc)
        return self._device.__exit__(*exc)


def _no_gradients(where, *tensors):
    """Refuses tensors whose gradients nobody works out: the result would be detached from them without a word."""
    import torch

    _no_tangents(where, *tensors)
    _check(not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors),
           f"{where} has no gradients: detach what requires one, or call it under torch.no_grad()")


def _no_tangents(where, *tensors):
    """Refuses tensors with a forward-mode derivative, which nobody works out."""
    from torch.autograd import forward_ad

    _check(all(t is None or forward_ad.unpack_dual(t).tangent is None for t in tensors), f"{where} has no forward-mode derivatives")


def _raise(rc, where):
    if rc != FLASH_OK:
        raise FlashError(rc, where)


def _written(*tensors):
    """Tells autograd that the caller's tensors have been written, so that a backward pass that has saved one of them notices."""
    import torch

    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


# ---------------------------------------------------------------------------------------------------- rotary positions


def rotary_frequencies(rot, base=10000.0, scaling=None, stretch=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0, device=None):
    """(inv_freq, factor) for flash_rotary: fp32 [rot / 2] with inv_freq[i] = base^(-2 i / rot), and the factor of the outputs.

    scaling lowers the frequencies for contexts `stretch` times longer than those that a model was trained on:
      None      as they are
      "linear"  all by stretch (positions are interpolated)
      "ntk"     base grows by stretch^(rot / (rot - 2)): the highest frequency stays, the lowest is divided by stretch
      "yarn"    pair i turns r = original_length * inv_freq[i] / (2 pi) times within the trained length; those with r >= beta_fast stay, those with
                r <= beta_slow are divided by stretch, between the two the share of either is linear in r.  The factor is
                0.1 ln(stretch) + 1, which with Q and K both turned divides the softmax temperature by its square."""
    import torch

    _check(isinstance(rot, int) and rot >= 2 and rot % 2 == 0, "rot must be an even number")
    _check(math.isfinite(base) and base > 0 and math.isfinite(stretch) and stretch > 0, "base and stretch must be positive")
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    factor = 1.0
    if scaling == "ntk":
        _check(rot > 2, "ntk scaling needs rot > 2")
        base = base * stretch ** (rot / (rot - 2))
    inv = base ** (-i / rot)
    if scaling == "linear":
        inv = inv / stretch
    elif scaling == "yarn":
        _check(original_length is not None and original_length > 0, "yarn scaling needs original_length")
        _check(beta_fast > beta_slow, "beta_fast must be above beta_slow")
        turns = original_length * inv / (2.0 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
        inv = keep * inv + (1.0 - keep) * inv / stretch
        factor = 0.1 * math.log(stretch) + 1.0 if stretch > 1.0 else 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'yarn'")
    return inv.to(torch.float32).to(device), factor


def _rotary_dims(t):
    """(B, H, N, strides of batch, head and row) of [B,H,N,d] or [N,H,d]"""
    s = t.stride()
    if t.dim() == 4:
        return (*t.shape[:3], s[0], s[1], s[2])
    return (1, t.shape[1], t.shape[0], 0, s[1], s[0])


def _positions_ok(positions):
    import torch

    return positions.dtype in (torch.int32, torch.int64) and (positions.dim() == 0 or positions.shape[-1] <= 1 or positions.stride(-1) == 1)


def _rotary(x, positions, inv_freq, interleaved, factor, inverse, out, stream):
    import torch

    kinds = _types()
    _check(x.dim() in (3, 4), "x must be [B,H,N,d] or [tokens,H,d]")
    _check(x.dtype in kinds, "x must be fp16, bf16 or fp32")
    _check(x.shape[-1] >= 1 and (x.shape[-1] == 1 or x.stride(-1) == 1), "the last dimension of x must be contiguous")
    _check(max(x.shape) <= _INT_MAX, "x is too large")
    B, H, N, xb, xh, xn = _rotary_dims(x)
    _check(_positions_ok(positions), "positions must be int32 or int64 with a contiguous last dimension")
    _check(tuple(positions.shape) == (N,) or (x.dim() == 4 and tuple(positions.shape) == (B, N)), "positions must be [N] or, for [B,H,N,d], [B,N]")
    _check(inv_freq.dtype == torch.float32 and inv_freq.dim() == 1 and inv_freq.is_contiguous(), "inv_freq must be contiguous fp32 [rot / 2]")
    _check(1 <= inv_freq.numel() <= x.shape[-1] // 2, "inv_freq must have 1 ... d / 2 elements")
    _check(not torch.is_grad_enabled() or not inv_freq.requires_grad, "inv_freq gets no gradient: detach it")
    _check(not torch.is_grad_enabled() or out is None or not out.requires_grad, "out must not require a gradient")
    device = _same_device(x, positions, inv_freq, out)
    with _on(device, stream) as handle:
        y = out
        if y is None:
            y = torch.empty_like(x)  # (in x's order of dimensions, dense)
            if y.shape[-1] > 1 and y.stride(-1) != 1:
                y = torch.empty(x.shape, dtype=x.dtype, device=device)
        else:
            _check(y.shape == x.shape and y.dtype == x.dtype and (y.shape[-1] == 1 or y.stride(-1) == 1),
                   "out must have x's shape and type and a contiguous last dimension")
        p = RotaryParams()
        L = _lib()
        L.flash_rotary_params_init(C.byref(p))
        p.X, p.Y, p.dtype = x.data_ptr(), y.data_ptr(), kinds[x.dtype]
        p.B, p.H, p.N, p.d, p.rot = B, H, N, x.shape[-1], 2 * inv_freq.numel()
        p.x_batch, p.x_head, p.x_row = xb, xh, xn
        p.y_batch, p.y_head, p.y_row = _rotary_dims(y)[3:]
        p.positions, p.positions_64 = positions.data_ptr(), int(positions.dtype == torch.int64)
        p.positions_batch = positions.stride(0) if positions.dim() == 2 else 0
        p.inv_freq, p.factor = inv_freq.data_ptr(), float(factor)
        p.interleaved, p.inverse = int(bool(interleaved)), int(bool(inverse))
        _raise(L.flash_rotary(C.byref(p), handle), "flash_rotary")
    _written(out)
    return y


def _rotary_function():
    import torch

    class Rotary(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, positions, inv_freq, interleaved, factor, inverse, stream):
            ctx.save_for_backward(positions, inv_freq)
            ctx.how = (interleaved, factor, inverse)
            return flash_rotary(x, positions, inv_freq, interleaved, factor, inverse, stream=stream)  # (no gradients in here)

        @staticmethod
        def backward(ctx, g):
            interleaved, factor, inverse = ctx.how
            positions, inv_freq = ctx.saved_tensors
            if g.shape[-1] > 1 and g.stride(-1) != 1:
                g = g.contiguous()
            return flash_rotary(g, positions, inv_freq, interleaved, factor, not inverse), None, None, None, None, None, None

    return Rotary


_function = None


def flash_rotary(x, positions, inv_freq, interleaved=False, factor=1.0, inverse=False, out=None, stream=None):
    """factor * R(position) x on the leading rot = 2 * inv_freq.numel() elements of every row, x itself behind them.

    x [B,H,N,d] with positions [N] or [B,N], or [tokens,H,d] with positions [tokens]; fp16, bf16 or fp32, any strides with a contiguous last
    dimension.  Pairs are (i, i + rot / 2), or (2 i, 2 i + 1) if interleaved.  inverse turns the other way: the gradient of x from the
    gradient of the result, which is also what backward() takes for an x that requires one.  out: where to, x itself for in place."""
    global _function
    if stream is None:
        y = (_native or _front_end()).rotary(x, positions, inv_freq, interleaved, factor, inverse, out)
        if y is not NotImplemented:
            return y
    # arguments that the native front end leaves alone (those that raise among them)
    import torch

    _no_tangents("flash_rotary", x, inv_freq, out)
    if torch.is_grad_enabled() and x.requires_grad:
        _check(out is None, "out cannot be given for an x that requires a gradient")
        _check(not inv_freq.requires_grad, "inv_freq gets no gradient: detach it")
        if _function is None:
            _function = _rotary_function()
        return _function.apply(x, positions, inv_freq, interleaved, factor, inverse, stream)
    return _rotary(x, positions, inv_freq, interleaved, factor, inverse, out, stream)


# ---------------------------------------------------------------------------------------------------- paged cache


def _rows(t, name, heads, d, dtype, tokens=None):
    _check(t.dim() == 3 and t.shape[1] == heads and t.shape[2] == d and (tokens is None or t.shape[0] == tokens),
           f"{name} must be [tokens,H,d] with the heads and head dimension of the call")
    _check(t.dtype == dtype, f"{name} must have the caches' type")
    _check(t.stride(2) == 1, f"the last dimension of {name} must be contiguous")
    return (t.stride(0), t.stride(1))


def _paged_params(k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, H, total_q):
    import torch

    kinds = _types()
    _check(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "k_cache and v_cache must be [pages,H_kv,page_size,d]")
    _check(k_cache.dtype in (torch.float16, torch.bfloat16) and v_cache.dtype == k_cache.dtype, "caches must be fp16 or bf16")
    _check(k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "the last dimension of the caches must be contiguous")
    for t, name, dim in ((block_table, "block_table", 2), (seqlens_k, "seqlens_k", 1), (cu_seqlens_q, "cu_seqlens_q", 1)):
        _check(t.dtype == torch.int32 and t.dim() == dim and (t.numel() == 0 or t.shape[-1] == 1 or t.stride(-1) == 1),
               f"{name} must be int32 with {dim} dimension(s), the last contiguous")
    B = seqlens_k.shape[0]
    _check(block_table.shape[0] == B and cu_seqlens_q.shape[0] == B + 1, "block_table, seqlens_k and cu_seqlens_q must be [B,pages], [B] and [B + 1]")
    _check(max(*k_cache.shape, *block_table.shape, total_q, H) <= _INT_MAX, "tensors are too large")
    p = PagedParams()
    _lib().flash_paged_params_init(C.byref(p))
    p.K_cache, p.V_cache, p.dtype = k_cache.data_ptr(), v_cache.data_ptr(), kinds[k_cache.dtype]
    p.block_table, p.seqlens_k, p.cu_seqlens_q = block_table.data_ptr(), seqlens_k.data_ptr(), cu_seqlens_q.data_ptr()
    p.num_pages, p.H_kv, p.page_size, p.d = k_cache.shape
    p.B, p.H, p.total_q, p.max_pages = B, H, total_q, block_table.shape[1]
    p.kc_page, p.kc_head, p.kc_row = k_cache.stride()[:3]
    p.vc_page, p.vc_head, p.vc_row = v_cache.stride()[:3]
    p.block_table_stride = block_table.stride(0)
    return p


def flash_append_paged(k, v, k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, q=None, inv_freq=None, interleaved=False, factor=1.0,
                       positions=None, out=None, stream=None):
    """Writes the new rows k, v [tokens,H_kv,d] into the sequences' pages, the last ones of seqlens_k keys each.

    With inv_freq K is turned on its way in as by flash_rotary, by its place in the sequence or by positions [tokens] where they are given, and
    so is q [tokens,H,d], if it is given: returned, in `out` if that is given (q itself for in place).  Returns None without q.  For serving: tensors
    that require a gradient are refused while gradients are recorded."""
    if stream is None:
        res = (_native or _front_end()).append(k, v, k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, q, inv_freq, interleaved, factor, positions, out)
        if res is not NotImplemented:
            return res
    # arguments that the native front end leaves alone (those that raise among them)
    import torch

    _no_gradients("flash_append_paged", k, v, k_cache, v_cache, q, inv_freq, out)
    _check(q is None or inv_freq is not None, "q is turned with inv_freq: without it there is nothing to do for q")
    _check(out is None or q is not None, "out is for q")
    _check(positions is None or inv_freq is not None, "positions are for inv_freq")
    _check(k.dim() == 3 and k_cache.dim() == 4 and (q is None or q.dim() == 3), "q, k and v must be [tokens,H,d], caches [pages,H_kv,page_size,d]")
    Hk, d = k_cache.shape[1], k_cache.shape[3]
    T = k.shape[0]
    p = _paged_params(k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, Hk if q is None else q.shape[1], T)
    p.k_token, p.k_head = _rows(k, "k", Hk, d, k_cache.dtype)
    p.v_token, p.v_head = _rows(v, "v", Hk, d, k_cache.dtype, T)
    p.K, p.V = k.data_ptr(), v.data_ptr()
    if inv_freq is not None:
        _check(inv_freq.dtype == torch.float32 and inv_freq.dim() == 1 and inv_freq.is_contiguous(), "inv_freq must be contiguous fp32 [rot / 2]")
        _check(1 <= inv_freq.numel() <= d // 2, "inv_freq must have 1 ... d / 2 elements")
        p.inv_freq, p.rot, p.interleaved, p.factor = inv_freq.data_ptr(), 2 * inv_freq.numel(), int(bool(interleaved)), float(factor)
    if positions is not None:
        _check(positions.dim() == 1 and positions.shape[0] == T and _positions_ok(positions), "positions must be int32 or int64 [tokens]")
        p.positions, p.positions_64 = positions.data_ptr(), int(positions.dtype == torch.int64)
    device = _same_device(k, v, k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, q, inv_freq, positions, out)
    given = out
    with _on(device, stream) as handle:
        if q is not None:
            p.q_token, p.q_head = _rows(q, "q", p.H, d, k_cache.dtype, T)
            if out is None:
                out = torch.empty(q.shape, dtype=q.dtype, device=device)
            p.o_token, p.o_head = _rows(out, "out", p.H, d, k_cache.dtype, T)
            p.Q, p.O = q.data_ptr(), out.data_ptr()
        _raise(_lib().flash_append_paged(C.byref(p), handle), "flash_append_paged")
    _written(k_cache, v_cache, given)
    return out


def flash_forward_paged(q, k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, max_seqlen_q=0, max_seqlen_k=0, softmax_scale=None, causal=False,
                        window=(-1, -1), num_splits=0, workspace=None, out=None, lse=None, stream=None, softcap=0.0, alibi_slopes=None, prefix_lens=None,
                        tree_mask=None):
    """Attention of the new tokens q [tokens,H,d] over their sequences' pages: (O [tokens,H,d], LSE fp32 [tokens,H]).

    Query head h reads K/V head h / (H / H_kv).  Token i of n stands at position seqlens_k - n + i; causal and window (left, right) are as in
    flash_forward, from there.  max_seqlen_q: at least the longest chunk of the call (0: the number of tokens), otherwise rows may be
    missing or meaningless; max_seqlen_k: the longest sequence, which decides into how many splits its keys are cut (0: what the table can name).
    num_splits <= 0: the library's choice.
    workspace: (O_partial, LSE_partial) of at least the bytes that paged_workspace_bytes says, otherwise allocated here.
    Rows that belong to no sequence are left as they are (new memory where out and lse are not given).  For serving: tensors that require a gradient
    are refused while gradients are recorded.

    softcap > 0: scores x become softcap * tanh(x / softcap), from FLASH_MIN_SOFTCAP to FLASH_MAX_SOFTCAP.  alibi_slopes: fp32 [H], from
    -FLASH_MAX_SLOPE to FLASH_MAX_SLOPE (device memory: not checked), score -= slope[h] * |i - j| of the positions, behind the cap.  prefix_lens:
    int32 [B], keys in front of it are seen by all of a sequence's tokens, whatever causal and a right window say.  tree_mask: int64 [tokens, words]
    (flash_tree_mask): bit j % 64 of word j / 64 says whether a token sees new token j of its sequence, in place of causal; with it max_seqlen_q is at
    most 64 * words, tokens stand at the chunk's begin plus their depth (bits less one), a right window and a prefix are refused, and a left window
    must reach over a chunk."""
    if stream is None:
        native = _native or _front_end()
        if softcap == 0 and alibi_slopes is None and prefix_lens is None and tree_mask is None:
            res = native.paged(q, k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, max_seqlen_q, max_seqlen_k, softmax_scale, causal, window,
                               num_splits, workspace, out, lse)
        else:
            res = native.paged(q, k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, max_seqlen_q, max_seqlen_k, softmax_scale, causal, window,
                               num_splits, workspace, out, lse, softcap, alibi_slopes, prefix_lens, tree_mask)
        if res is not NotImplemented:
            return res
    # arguments that the native front end leaves alone (those that raise among them)
    import torch

    _no_gradients("flash_forward_paged", q, k_cache, v_cache, out, lse, alibi_slopes)
    _check(q.dim() == 3 and k_cache.dim() == 4, "q must be [tokens,H,d], caches [pages,H_kv,page_size,d]")
    T, H, d = q.shape
    Hk = k_cache.shape[1]
    _check(Hk >= 1 and H >= 1 and H % Hk == 0, "H must be a multiple of H_kv")
    p = _paged_params(k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, H, T)
    p.q_token, p.q_head = _rows(q, "q", H, k_cache.shape[3], k_cache.dtype)
    p.Q = q.data_ptr()
    p.max_seqlen_q, p.max_seqlen_k = _int(max_seqlen_q), _int(max_seqlen_k)
    p.softmax_scale = float(softmax_scale) if softmax_scale is not None else d ** -0.5
    p.is_causal = int(bool(causal))
    p.window_left, p.window_right = _int(window[0]), _int(window[1])
    p.num_splits = _int(num_splits)
    p.softcap = float(softcap)
    if alibi_slopes is not None:
        _check(alibi_slopes.dtype == torch.float32 and tuple(alibi_slopes.shape) == (H,) and alibi_slopes.is_contiguous(), "alibi_slopes must be contiguous fp32 [H]")
        p.alibi_slopes = alibi_slopes.data_ptr()
    if prefix_lens is not None:
        _check(prefix_lens.dtype == torch.int32 and tuple(prefix_lens.shape) == (p.B,) and prefix_lens.is_contiguous(), "prefix_lens must be contiguous int32 [B]")
        p.prefix_lens = prefix_lens.data_ptr()
    if tree_mask is not None:
        p.tree_words, p.tree_stride = _tree_rows(tree_mask, T)
        p.tree_mask = tree_mask.data_ptr()
        _check(T == 0 or tree_mask.data_ptr() != 0, "tree_mask is empty")
    given = workspace if workspace is not None else ()
    device = _same_device(q, k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, out, lse, alibi_slopes, prefix_lens, tree_mask, *given)
    L = _lib()
    S = L.flash_forward_paged_resolve_splits(C.byref(p))
    if S < 0:
        raise FlashError(S, "flash_forward_paged_resolve_splits")
    rows = T * H * S if S > 1 else 0
    with _on(device, stream) as handle:
        o = out if out is not None else torch.empty((T, H, d), dtype=q.dtype, device=device)
        p.o_token, p.o_head = _rows(o, "out", H, d, q.dtype, T)
        l = lse if lse is not None else torch.empty((T, H), dtype=torch.float32, device=device)
        _check(l.dtype == torch.float32 and tuple(l.shape) == (T, H) and l.is_contiguous(), "lse must be contiguous fp32 [tokens,H]")
        p.O, p.LSE = o.data_ptr(), l.data_ptr()
        if rows and workspace is None:
            workspace = (torch.empty(rows * d, dtype=torch.float32, device=device), torch.empty(rows, dtype=torch.float32, device=device))
        if workspace is not None:
            _check(len(workspace) == 2 and all(t.dtype == torch.float32 and t.is_contiguous() for t in workspace),
                   "workspace must be two contiguous fp32 tensors")
            _check(workspace[0].numel() >= rows * d and workspace[1].numel() >= rows,
                   f"workspace too small for {S} splits: need {rows * d} and {rows} fp32 elements")
            p.O_partial, p.LSE_partial = workspace[0].data_ptr(), workspace[1].data_ptr()
        _raise(L.flash_forward_paged(C.byref(p), handle), "flash_forward_paged")
    _written(out, lse, *given)
    return o, l


def _tree_rows(mask, tokens):
    """(words, stride) of a mask [tokens, words]"""
    import torch

    _check(mask.dtype == torch.int64 and mask.dim() == 2 and mask.shape[0] == tokens and 1 <= mask.shape[1] <= FLASH_MAX_TREE_TOKENS // 64,
           f"a tree's mask must be int64 [tokens,words] with 1 ... {FLASH_MAX_TREE_TOKENS // 64} words")
    _check(mask.shape[1] == 1 or mask.stride(1) == 1, "the last dimension of a tree's mask must be contiguous")
    return mask.shape[1], max(mask.stride(0), mask.shape[1]) if tokens <= 1 else mask.stride(0)


def flash_tree_mask(parents, cu_seqlens_q, seqlens_k=None, max_seqlen_q=0, mask=None, positions=None, stream=None):
    """(mask int64 [tokens, words], positions int32 [tokens]) of the trees whose tokens have these parents, int32 [tokens], numbered within their chunk.

    A parent stands in front of its children; a number that is not below the token's own, or negative, says that it has none and hangs on the keys in
    front of the chunk.  A token's row has the bits of the tokens on its path, its own among them, and it stands at seqlens_k - n + (tokens on the
    path) - 1, without seqlens_k counted from the chunk's begin.  max_seqlen_q: at least the longest chunk (0: the number of tokens), which
    decides the words, 64 tokens each, up to FLASH_MAX_TREE_TOKENS.  mask, positions: where to; rows of no sequence are left as they are (new memory
    where these are not given)."""
    if stream is None:
        res = (_native or _front_end()).tree_mask(parents, cu_seqlens_q, seqlens_k, max_seqlen_q, mask, positions)
        if res is not NotImplemented:
            return res
    import torch

    for t, name in ((parents, "parents"), (cu_seqlens_q, "cu_seqlens_q"), (seqlens_k, "seqlens_k")):
        _check(t is None or (t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous()), f"{name} must be contiguous int32 with one dimension")
    T, B = parents.shape[0], cu_seqlens_q.shape[0] - 1
    _check(B >= 0 and (seqlens_k is None or seqlens_k.shape[0] == B), "cu_seqlens_q and seqlens_k must be [B + 1] and [B]")
    _check(max(T, B) <= _INT_MAX, "tensors are too large")
    most = min(T, max_seqlen_q) if max_seqlen_q > 0 else T
    _check(most <= FLASH_MAX_TREE_TOKENS, f"trees have at most {FLASH_MAX_TREE_TOKENS} tokens (max_seqlen_q)")
    words = max(1, -(-most // 64))
    device = _same_device(parents, cu_seqlens_q, seqlens_k, mask, positions)
    given = (mask, positions)
    with _on(device, stream) as handle:
        if mask is None:
            mask = torch.empty((T, words), dtype=torch.int64, device=device)
        if positions is None:
            positions = torch.empty(T, dtype=torch.int32, device=device)
        p = TreeParams()
        p.words, p.mask_stride = _tree_rows(mask, T)
        _check(p.words >= words, "mask has too few words")
        _check(positions.dtype == torch.int32 and tuple(positions.shape) == (T,) and positions.is_contiguous(), "positions must be contiguous int32 [tokens]")
        p.parents, p.cu_seqlens_q, p.mask, p.positions = parents.data_ptr(), cu_seqlens_q.data_ptr(), mask.data_ptr(), positions.data_ptr()
        p.seqlens_k = seqlens_k.data_ptr() if seqlens_k is not None else None
        p.B, p.total_q = B, T
        _raise(_lib().flash_tree_mask(C.byref(p), handle), "flash_tree_mask")
    _written(*given)
    return mask, positions


def flash_keep_paged(k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, path, accepted, out=None, stream=None):
    """Moves the rows of the accepted path of each sequence's drafted tokens to the places behind the keys in front of them; returns the lengths, int32 [B].

    Caches [pages,H_kv,page_size,d], or [layers,pages,H_kv,page_size,d] for all layers at once.  path: int32 [B, L], the path's tokens by their numbers in
    the chunk, which grow; accepted: int32 [B], how many of them stay.  Row path[b, i] of the chunk goes to its row i; a path ends in front of the
    first number that does not grow or is not a token of the chunk.  Returned: seqlens_k - n + tokens that stay, in `out` if that is given, which cannot
    lie in one of the other index tensors."""
    if stream is None:
        res = (_native or _front_end()).keep(k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, path, accepted, out)
        if res is not NotImplemented:
            return res
    import torch

    _no_gradients("flash_keep_paged", k_cache, v_cache)
    _check(k_cache.dim() in (4, 5) and k_cache.shape == v_cache.shape, "k_cache and v_cache must be [pages,H_kv,page_size,d] or [layers,pages,H_kv,page_size,d]")
    many = k_cache.dim() == 5
    _check(k_cache.dtype in (torch.float16, torch.bfloat16) and v_cache.dtype == k_cache.dtype, "caches must be fp16 or bf16")
    _check(k_cache.stride(-1) == 1 and v_cache.stride(-1) == 1, "the last dimension of the caches must be contiguous")
    for t, name, dim in ((block_table, "block_table", 2), (path, "path", 2), (seqlens_k, "seqlens_k", 1), (cu_seqlens_q, "cu_seqlens_q", 1), (accepted, "accepted", 1),
                         (out, "out", 1)):
        _check(t is None or (t.dtype == torch.int32 and t.dim() == dim and (t.numel() == 0 or t.shape[-1] == 1 or t.stride(-1) == 1)),
               f"{name} must be int32 with {dim} dimension(s), the last contiguous")
    B = seqlens_k.shape[0]
    _check(block_table.shape[0] == B and path.shape[0] == B and accepted.shape[0] == B and cu_seqlens_q.shape[0] == B + 1 and (out is None or out.shape[0] == B),
           "block_table, path, accepted, seqlens_k and cu_seqlens_q must be [B,pages], [B,L], [B], [B] and [B + 1]")
    _check(max(*k_cache.shape, *block_table.shape, *path.shape) <= _INT_MAX, "tensors are too large")
    device = _same_device(k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, path, accepted, out)
    given = out
    with _on(device, stream) as handle:
        if out is None:
            out = torch.empty(B, dtype=torch.int32, device=device)
        p = KeepParams()
        p.K_cache, p.V_cache = k_cache.data_ptr(), v_cache.data_ptr()
        p.block_table, p.seqlens_k, p.cu_seqlens_q = block_table.data_ptr(), seqlens_k.data_ptr(), cu_seqlens_q.data_ptr()
        p.path, p.accepted, p.seqlens_out = path.data_ptr(), accepted.data_ptr(), out.data_ptr()
        p.num_pages, p.H_kv, p.page_size, p.d = k_cache.shape[-4:]
        p.B, p.layers, p.max_pages, p.max_path = B, k_cache.shape[0] if many else 1, block_table.shape[1], path.shape[1]
        p.kc_page, p.kc_head, p.kc_row = k_cache.stride()[-4:-1]
        p.vc_page, p.vc_head, p.vc_row = v_cache.stride()[-4:-1]
        if many:
            p.kc_layer, p.vc_layer = k_cache.stride(0), v_cache.stride(0)
        if p.layers == 0:  # (the lengths alone: one layer without pages)
            p.layers, p.num_pages = 1, 0
        p.block_table_stride, p.path_stride = block_table.stride(0), path.stride(0)
        _raise(_lib().flash_keep_paged(C.byref(p), handle), "flash_keep_paged")
    _written(k_cache, v_cache, given)
    return out


def _paged_shape(B, H, H_kv, d, total_q, page_size, max_pages, max_seqlen_q, max_seqlen_k, causal, window, num_splits, softcap, alibi, prefix, tree_words):
    _check(max(B, H, H_kv, d, total_q, page_size, max_pages) <= _INT_MAX, "sizes are too large")
    p = PagedParams()
    _lib().flash_paged_params_init(C.byref(p))
    p.B, p.H, p.H_kv, p.d, p.total_q, p.page_size, p.max_pages = B, H, H_kv, d, total_q, page_size, max_pages
    p.num_pages = 1
    p.max_seqlen_q, p.max_seqlen_k = _int(max_seqlen_q), _int(max_seqlen_k)
    p.is_causal, p.window_left, p.window_right, p.num_splits = int(bool(causal)), _int(window[0]), _int(window[1]), _int(num_splits)
    p.softcap = float(softcap)
    # (only whether they are there matters)
    if alibi:
        p.alibi_slopes = 16
    if prefix:
        p.prefix_lens = 16
    if tree_words:
        p.tree_mask, p.tree_words, p.tree_stride = 16, _int(tree_words), _int(tree_words)
    return p


def paged_resolve_splits(B, H, H_kv, d, total_q, page_size, max_pages, max_seqlen_q=0, max_seqlen_k=0, causal=False, window=(-1, -1), num_splits=0,
                         softcap=0.0, alibi=False, prefix=False, tree_words=0):
    """The split count that flash_forward_paged will use for such a call.  alibi, prefix: whether it has alibi_slopes, prefix_lens; tree_words: of its
    tree_mask."""
    S = _lib().flash_forward_paged_resolve_splits(C.byref(_paged_shape(B, H, H_kv, d, total_q, page_size, max_pages, max_seqlen_q, max_seqlen_k,
                                                                       causal, window, num_splits, softcap, alibi, prefix, tree_words)))
    if S < 0:
        raise FlashError(S, "flash_forward_paged_resolve_splits")
    return S


def paged_workspace_bytes(B, H, H_kv, d, total_q, page_size, max_pages, max_seqlen_q=0, max_seqlen_k=0, causal=False, window=(-1, -1), num_splits=0,
                          softcap=0.0, alibi=False, prefix=False, tree_words=0):
    """Bytes of (O_partial, LSE_partial) for flash_forward_paged calls of these sizes and masks."""
    ob, lb = C.c_size_t(), C.c_size_t()
    _raise(_lib().flash_forward_paged_workspace_bytes(C.byref(_paged_shape(B, H, H_kv, d, total_q, page_size, max_pages, max_seqlen_q, max_seqlen_k,
                                                                           causal, window, num_splits, softcap, alibi, prefix, tree_words)), C.byref(ob), C.byref(lb)),
           "flash_forward_paged_workspace_bytes")
    return ob.value, lb.value
