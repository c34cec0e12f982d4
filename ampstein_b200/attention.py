"""Operators between the q|k|v projections and o: rotary positions with the write into a paged key-value cache (rope,
rope_append), attention over that cache (paged_attention), copies of its pages (copy_pages). The reference runs kernels of its
own there over contiguous caches (src/ucode/ampstein/graphdec.uc:171-190); these are this library's, with one interface for
prompts, drafted and single tokens.

Common to rope, rope_append and paged_attention: a row of q is a token. pos (seqs) int32 or int64 holds the position of every
sequence's first token of the call. Without cu all sequences have rows / seqs tokens; with cu (seqs + 1 int32, ascending) sequence b
has rows cu[b] .. cu[b + 1] - 1, and rows behind cu[seqs] are left as they were. A token at a negative position belongs to no
sequence (an unused slot of a captured batch): it is rotated, not stored, and its attention is 0.

Caches are (pages, page_size, kv_heads, dim), with any strides but the last (a cache kept per head is passed as its transpose);
table (seqs, max_pages) int32 names the pages of each sequence. Every call runs on the current stream of q's device, allocates its
workspace with torch (each captured graph has its own), and never synchronises.
"""
import functools
import math
import struct
from array import array

import torch

from . import _lib
from .exl3 import _launch

_DTYPES = (torch.float16, torch.bfloat16)
WIDTHS = (64, 128, 256)                # values per head that paged_attention takes
_MAX_POS = 1 << 30                     # positions of one sequence

_ROPE = struct.Struct("=10q15q12if4x")             # amp_rope_args
_ATTENTION = struct.Struct("=10q11q12if4x")        # amp_attention_args


_direct = None                         # the calls of csrc_py/tensor_call.h by name; {} where torch has no table for them


def _calls():
    global _direct
    _lib.lib()
    from . import _fast
    names = ("rope_call", "attention_call", "copy_call")
    _direct = {n: getattr(_fast, n) for n in names} if hasattr(_fast, "tensor_setup") and _fast.tensor_setup(torch.Tensor) else {}
    return _direct


def _cuda(name, what, t, dev=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s: %s must be a torch tensor" % (name, what))
    if not t.is_cuda:
        raise RuntimeError("%s: tensors must live on a CUDA device (no CPU path exists); %s does not" % (name, what))
    if dev is not None and t.get_device() != dev:
        raise ValueError("%s: %s is on another device" % (name, what))


def _rows(name, what, t, dtype, dev, shape=None):
    """Strides (row, head) of a (rows, heads, dim) tensor"""
    _cuda(name, what, t, dev)
    if t.dtype != dtype:
        raise TypeError("%s: %s must be %s" % (name, what, dtype))
    if t.dim() != 3 or (shape is not None and tuple(t.shape) != shape):
        raise ValueError("%s: %s must be (rows, heads, dim)%s" % (name, what, " = %s" % (shape,) if shape is not None else ""))
    n, h, d = t.shape
    s = t.stride()
    if d > 1 and s[2] != 1:
        raise ValueError("%s: the values of a head of %s must be contiguous" % (name, what))
    return (s[0] if n > 1 else 0), (s[1] if h > 1 else 0)


def _cache(name, what, t, dtype, dev, shape):
    """Strides (page, row, head) of a (pages, page_size, kv_heads, dim) tensor"""
    _cuda(name, what, t, dev)
    if t.dtype != dtype:
        raise TypeError("%s: %s must be %s, as q" % (name, what, dtype))
    if t.dim() != 4 or (shape is not None and tuple(t.shape) != shape):
        raise ValueError("%s: both caches must be (pages, page_size, kv_heads, dim) of one shape" % name)
    s, z = t.stride(), t.shape
    if z[3] > 1 and s[3] != 1:
        raise ValueError("%s: the values of a head of %s must be contiguous" % (name, what))
    return tuple(s[i] if z[i] > 1 else 0 for i in range(3))


def _apart(name, what, t):
    """Whether what is written lies at places of its own: no stride inside the extent of a smaller one"""
    extent = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if st < extent:
            raise ValueError("%s: places of %s overlap" % (name, what))
        extent = st * (n - 1) + extent


def _span(t):
    """First byte, and [(size, stride in bytes)] of a tensor's dimensions that go somewhere"""
    z = t.element_size()
    return t.data_ptr(), [(n, st * z) for n, st in zip(t.shape, t.stride()) if n > 1 and st], z


def _extent(dims, period, z):
    return z + sum((n - 1) * st for n, st in dims if not period or st % period)


def _share(t, u):
    """Whether two tensors may share memory: their extents meet, and do so round each of their strides as well (columns of one buffer,
    or keys and values side by side in a page, do not share any)"""
    if t.numel() == 0 or u.numel() == 0:
        return False
    (a, da, za), (b, db, zb) = _span(t), _span(u)
    if a + _extent(da, 0, za) <= b or b + _extent(db, 0, zb) <= a:
        return False
    for _, p in da + db:
        ea, eb, d = _extent(da, p, za), _extent(db, p, zb), (b - a) % p
        if d >= ea and d + eb <= p:
            return False
    return True


def _not_shared(name, what, t, others):
    for which, u in others:
        if u is not None and _share(t, u):
            raise ValueError("%s: %s overlaps %s" % (name, what, which))


def _sequences(name, rows, pos, cu, dev):
    _cuda(name, "pos", pos, dev)
    if pos.dtype not in (torch.int32, torch.int64) or pos.dim() != 1 or not pos.is_contiguous():
        raise TypeError("%s: pos must be int32 or int64, one contiguous value per sequence" % name)
    seqs = pos.shape[0]
    if cu is not None:
        _cuda(name, "cu", cu, dev)
        if cu.dtype != torch.int32 or cu.dim() != 1 or not cu.is_contiguous() or cu.shape[0] != seqs + 1:
            raise TypeError("%s: cu must be int32, one contiguous value per sequence and one more" % name)
    elif (rows % seqs if seqs else rows):
        raise ValueError("%s: %d rows do not divide into %d sequences (cu says how)" % (name, rows, seqs))
    return seqs


def _table(name, table, seqs, page_size, dev):
    _cuda(name, "table", table, dev)
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != seqs or (table.shape[1] > 1 and table.stride(1) != 1):
        raise TypeError("%s: table must be (seqs, max_pages) int32 with contiguous rows" % name)
    if table.shape[1] * page_size > _MAX_POS:
        raise ValueError("%s: more than 2^30 positions per sequence" % name)
    return table.shape[1], (table.stride(0) if seqs > 1 else 0)


def rope_frequencies(rot, theta=10000.0, scaling=None, device="cuda"):
    """(inv_freq, mscale) for rope / rope_append: inv_freq (rot / 2) float32 on `device`, mscale a float. scaling: None, or a dict
    with "kind" and a "factor" s:
      "linear"  positions divided by s
      "ntk"     theta multiplied by s^(rot / (rot - 2)): fast dimensions keep their angle, slow ones are stretched
      "llama3"  wavelengths longer than original / low_freq_factor divided by s, shorter than original / high_freq_factor kept, a linear
                mix between; "original" positions (8192), "low_freq_factor" (1), "high_freq_factor" (4)
      "yarn"    dimensions that turn more than beta_fast times over the original positions kept, fewer than beta_slow times divided
                by s, a linear mix between; mscale = "attention_factor", or 0.1 ln s + 1; "original" (4096), "beta_fast" (32),
                "beta_slow" (1)"""
    if rot <= 0 or rot % 2:
        raise ValueError("rope_frequencies: rot must be even and positive, not %s" % (rot,))
    if not theta > 0:
        raise ValueError("rope_frequencies: theta must be positive, not %s" % (theta,))
    opts = dict(scaling or {})
    kind = opts.pop("kind", "none")
    factor = float(opts.pop("factor", 1.0))
    names = {"none": (), "linear": (), "ntk": (), "llama3": ("original", "low_freq_factor", "high_freq_factor"),
             "yarn": ("original", "beta_fast", "beta_slow", "attention_factor")}
    if kind not in names:
        raise ValueError("rope_frequencies: unknown scaling %r (%s)" % (kind, ", ".join(names)))
    if set(opts) - set(names[kind]):
        raise ValueError("rope_frequencies: %s scaling takes no %s" % (kind, ", ".join(sorted(set(opts) - set(names[kind])))))
    if not factor > 0 or not math.isfinite(factor):
        raise ValueError("rope_frequencies: factor must be positive, not %s" % factor)
    theta, mscale = float(theta), 1.0
    if kind == "ntk" and rot > 2:
        theta *= factor ** (rot / (rot - 2))
    freq = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    if kind == "linear":
        freq = [f / factor for f in freq]
    elif kind == "llama3":
        original, lo, hi = opts.get("original", 8192), opts.get("low_freq_factor", 1.0), opts.get("high_freq_factor", 4.0)
        if not original > 0 or not hi > lo:
            raise ValueError("rope_frequencies: original must be positive and high_freq_factor above low_freq_factor")
        for i, f in enumerate(freq):
            keep = min(1.0, max(0.0, (original * f / (2 * math.pi) - lo) / (hi - lo)))
            freq[i] = keep * f + (1 - keep) * f / factor
    elif kind == "yarn":
        original, fast, slow = opts.get("original", 4096), opts.get("beta_fast", 32.0), opts.get("beta_slow", 1.0)
        if not original > 0 or not fast > slow or not slow > 0 or not theta > 1:
            raise ValueError("rope_frequencies: original and beta_slow must be positive, beta_fast above beta_slow, theta above 1")
        # the dimension that turns r times over the original positions
        turning = lambda r: rot * math.log(original / (r * 2 * math.pi)) / (2 * math.log(theta))      # noqa: E731
        low, high = max(0, math.floor(turning(fast))), min(rot - 1, math.ceil(turning(slow)))
        for i, f in enumerate(freq):
            keep = 1 - min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            freq[i] = keep * f + (1 - keep) * f / factor
        mscale = opts.get("attention_factor")
        mscale = float(mscale) if mscale is not None else (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
    return torch.tensor(freq, dtype=torch.float32, device=device), mscale


def _rope(name, q, kv, pos, inv_freq, cu, interleaved, mscale, out):
    call = (_calls() if _direct is None else _direct).get("rope_call")
    if call is not None and type(q) is torch.Tensor:
        k, v, kc, vc, table = kv or (None,) * 5
        y = q.new_empty(q.shape) if out is None else out
        if call(q, k, v, pos, inv_freq, kc, vc, table, cu, interleaved, mscale, y) is not None:
            return y
    _cuda(name, "q", q)
    dev, dtype = q.get_device(), q.dtype
    if dtype not in _DTYPES:
        raise TypeError("%s: q must be float16 or bfloat16" % name)
    qs = _rows(name, "q", q, dtype, dev)
    rows, heads, dim = q.shape
    seqs = _sequences(name, rows, pos, cu, dev)
    _cuda(name, "inv_freq", inv_freq, dev)
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() or 2 * inv_freq.shape[0] > dim:
        raise ValueError("%s: inv_freq must be contiguous float32, one value per rotated pair (at most %d)" % (name, dim // 2))
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=dtype, device=q.device)
        os = (heads * dim, dim)
    else:
        os = _rows(name, "out", out, dtype, dev, (rows, heads, dim))
        _apart(name, "out", out)
        if (out.data_ptr() != q.data_ptr() or os != qs) and _share(out, q):
            raise ValueError("%s: out overlaps q (it may be q itself)" % name)
    if kv is None:
        k = v = kc = vc = table = None
        kv_heads = pages = page_size = max_pages = 0
        ks, vs, cs = (0, 0), (0, 0), (0,) * 7
    else:
        k, v, kc, vc, table = kv
        _cuda(name, "k", k, dev)
        ks = _rows(name, "k", k, dtype, dev)
        kv_heads = k.shape[1]
        if k.shape[0] != rows or k.shape[2] != dim:
            raise ValueError("%s: k and v must have q's rows and head width" % name)
        vs = _rows(name, "v", v, dtype, dev, (rows, kv_heads, dim))
        kcs = _cache(name, "k_cache", kc, dtype, dev, None)
        pages, page_size = kc.shape[:2]
        if tuple(kc.shape[2:]) != (kv_heads, dim) or pages < 1 or page_size < 1:
            raise ValueError("%s: the caches must be (pages, page_size, %d, %d)" % (name, kv_heads, dim))
        vcs = _cache(name, "v_cache", vc, dtype, dev, tuple(kc.shape))
        _apart(name, "k_cache", kc)
        _apart(name, "v_cache", vc)
        for what, t in (("out", out), ("k_cache", kc), ("v_cache", vc)):
            _not_shared(name, what, t, (("k", k), ("v", v)))
        _not_shared(name, "k_cache", kc, (("v_cache", vc), ("q", q), ("out", out)))
        _not_shared(name, "v_cache", vc, (("q", q), ("out", out)))
        max_pages, tr = _table(name, table, seqs, page_size, dev)
        cs = kcs + vcs + (tr,)
    if rows == 0 or seqs == 0:
        return out
    ptr = lambda t: 0 if t is None else t.data_ptr()                                                  # noqa: E731
    args = _ROPE.pack(q.data_ptr(), ptr(k), ptr(v), out.data_ptr(), ptr(kc), ptr(vc), ptr(table), pos.data_ptr(), ptr(cu), inv_freq.data_ptr(),
                      *qs, *ks, *vs, *os, *cs, rows, seqs, heads, kv_heads, dim, 2 * inv_freq.shape[0], 1 if interleaved else 0,
                      pages, page_size, max_pages,
                      1 if dtype is torch.bfloat16 else 0, 1 if pos.dtype is torch.int64 else 0, mscale)
    _launch(q, "amp_b200_rope", args)
    return out


def rope(q, pos, inv_freq, cu=None, interleaved=False, mscale=1.0, out=None):
    """Rotary positions: the first 2 * len(inv_freq) values of every head of q (rows, heads, dim) turn in pairs (i, i + len(inv_freq)),
    or (2 i, 2 i + 1) with interleaved, by position * inv_freq[i]; cos and sin are multiplied by mscale. fp16 or bf16, any even
    number of rotated values, heads up to 1024 wide. The angle is taken modulo a turn in fp64 (off by less than 2^-21 at positions up to
    2^30), then rounded to fp32 (pi 2^-24); the turn is made in fp32 and rounded once.
    out: where to (it may be q itself, but must not overlap it otherwise). Returns out."""
    return _rope("rope", q, None, pos, inv_freq, cu, interleaved, mscale, out)


def rope_append(q, k, v, pos, inv_freq, k_cache, v_cache, table, cu=None, interleaved=False, mscale=1.0, out=None):
    """rope of q and k, and the write of k (rotated) and v (rows, kv_heads, dim) into the caches' pages, in one launch: the token at
    position p goes to row p % page_size of page table[b][p / page_size]. A token before position 0, beyond the table or on a page
    outside the pool is not stored. Two tokens of a call must not have the same place; k, v and the caches must not overlap each other,
    nor q and out. Returns the rotated q; the rotated k is
    only in the cache."""
    return _rope("rope_append", q, (k, v, k_cache, v_cache, table), pos, inv_freq, cu, interleaved, mscale, out)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(dev, *sizes):
    with torch.cuda.device(dev):
        n = _lib.lib().amp_b200_attention_workspace(*sizes)
    if n < 0:
        raise _lib.AmpError("amp_b200_attention_workspace", n, _lib.last_error())
    return n


def paged_attention(q, k_cache, v_cache, table, pos, cu=None, window=0, sinks=0, scale=None, out=None, lse=None):
    """Attention of q (rows, heads, dim), fp16 or bf16, dim 64 / 128 / 256, over caches that hold the rows' own keys and values
    already (rope_append). The token at position p sees the keys at positions j <= p, with window > 0 only the last `window` of
    them (its own among them) and the first `sinks`. heads is a multiple of kv_heads; query head h reads key-value head
    h // (heads / kv_heads). scale: 1 / sqrt(dim) by default. Returns out (rows, heads, dim), q's type; lse (rows, heads) float32, if
    given, takes ln sum_j exp(scale * q . k_j). Neither must overlap the other, q or a cache.

    An infinite or NaN key or value reaches the tokens that see it, no others. A token that sees nothing, or whose scores are all -inf, gets 0 (lse -inf). Pages that no token of the call can see are not read, and their table entries may hold
    anything; a token with a visible key on a page outside the pool, or beyond the table, gets NaN. Single tokens, a few drafted ones and
    prompt chunks may be mixed in one call with cu."""
    name = "paged_attention"
    call = (_calls() if _direct is None else _direct).get("attention_call")
    if call is not None and type(q) is torch.Tensor:
        y = q.new_empty(q.shape) if out is None else out
        s = q.shape[-1] ** -0.5 if scale is None and q.shape and q.shape[-1] else scale
        n = call(q, k_cache, v_cache, table, pos, cu, window, sinks, s, y, lse, None)
        if n:
            n = call(q, k_cache, v_cache, table, pos, cu, window, sinks, s, y, lse, torch.empty(n, dtype=torch.uint8, device=q.device))
        if n == 0:
            return y
    _cuda(name, "q", q)
    dev, dtype = q.get_device(), q.dtype
    if dtype not in _DTYPES:
        raise TypeError("%s: q must be float16 or bfloat16" % name)
    qs = _rows(name, "q", q, dtype, dev)
    rows, heads, dim = q.shape
    seqs = _sequences(name, rows, pos, cu, dev)
    ks = _cache(name, "k_cache", k_cache, dtype, dev, None)
    shape = tuple(k_cache.shape)
    pages, page_size, kv_heads, width = shape
    if width != dim or pages < 1 or page_size < 1 or kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError("%s: incompatible shapes (q %s, cache %s)" % (name, tuple(q.shape), shape))
    if dim not in WIDTHS:
        raise ValueError("%s: head width %d (64, 128 or 256)" % (name, dim))
    vs = _cache(name, "v_cache", v_cache, dtype, dev, shape)
    max_pages, tr = _table(name, table, seqs, page_size, dev)
    if window < 0 or sinks < 0:
        raise ValueError("%s: window and sinks must not be negative" % name)
    scale = dim ** -0.5 if scale is None else float(scale)
    if not abs(scale) * math.log2(math.e) < 3.4e38:
        raise ValueError("%s: scale must be finite (in float32, as scores in powers of two)" % name)
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=dtype, device=q.device)
        os = (heads * dim, dim)
    else:
        os = _rows(name, "out", out, dtype, dev, (rows, heads, dim))
        _apart(name, "out", out)
        _not_shared(name, "out", out, (("q", q), ("k_cache", k_cache), ("v_cache", v_cache)))
    if lse is not None:
        _cuda(name, "lse", lse, dev)
        if lse.dtype != torch.float32 or tuple(lse.shape) != (rows, heads) or not lse.is_contiguous():
            raise ValueError("%s: lse must be contiguous float32 (rows, heads)" % name)
        _not_shared(name, "lse", lse, (("out", out), ("q", q), ("k_cache", k_cache), ("v_cache", v_cache)))
    if rows == 0 or seqs == 0:
        return out
    window, sinks = min(int(window), _MAX_POS), min(int(sinks), _MAX_POS)
    n = _workspace_bytes(dev, rows, seqs, heads, kv_heads, dim, 0 if cu is None else 1, max_pages * page_size, window, sinks)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    args = _ATTENTION.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                           table.data_ptr(), pos.data_ptr(), 0 if cu is None else cu.data_ptr(), 0 if ws is None else ws.data_ptr(), n,
                           *qs, *os, *ks, *vs, tr, rows, seqs, heads, kv_heads, dim, pages, page_size, max_pages,
                           window, sinks, 1 if dtype is torch.bfloat16 else 0,
                           1 if pos.dtype is torch.int64 else 0, scale)
    _launch(q, "amp_b200_attention", args)
    return out


def attention_status(device=None):
    """0; or 1, a bounded wait in a call of paged_attention with prompt chunks ran out since the last look, or 2, such a call got shared
    memory without the alignment that it needs: what depended on it was not stored. Waits for all streams of the device; refused while
    the current stream is being captured."""
    import ctypes
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("attention_status: waits for the device, which a capture does not allow")
    v = ctypes.c_int(0)
    with torch.cuda.device(device):
        _lib.call("amp_b200_attention_status", ctypes.byref(v))
    return v.value


def _page_list(what, xs):
    if isinstance(xs, torch.Tensor):
        if xs.is_cuda or xs.dim() != 1 or xs.dtype not in (torch.int32, torch.int64):
            raise TypeError("copy_pages: %s must be whole numbers on the host" % what)
        xs = xs.tolist()
    try:
        return array("i", xs)
    except (TypeError, OverflowError):
        raise TypeError("copy_pages: %s must be a list of page numbers" % what) from None


def copy_pages(caches, src, dst):
    """Page dst[i] := page src[i] in every cache of the list, in one launch (more for long lists): a fork's own copy of a page that
    others go on writing, the moves of a compaction. A cache is (pages, page_size, kv_heads, dim), or (layers, pages, page_size, kv_heads,
    dim) with all layers copied; all of one shape and type on one device, and a page must be without gaps. src and dst are host lists. A
    page outside the pool, a page written twice and a page that is both read and written by different copies are refused. Returns
    caches."""
    name = "copy_pages"
    call = (_calls() if _direct is None else _direct).get("copy_call")
    if call is not None and call(caches, src, dst) == 0:
        return caches
    src, dst = _page_list("src", src), _page_list("dst", dst)
    if len(src) != len(dst):
        raise ValueError("%s: %d sources for %d destinations" % (name, len(src), len(dst)))
    if not caches:
        return caches
    first = caches[0]
    _cuda(name, "cache", first)
    dev, shape, size = first.get_device(), first.shape, first.element_size()
    if first.dim() not in (4, 5):
        raise ValueError("%s: caches must be (pages, page_size, kv_heads, dim), or with a layer dimension in front" % name)
    lead = first.dim() - 4
    inside = shape[lead + 1:]
    count = inside[0] * inside[1] * inside[2]
    ptrs, layer, page = array("Q"), array("q"), array("q")
    for t in caches:
        _cuda(name, "cache", t, dev)
        if t.shape != shape or t.dtype != first.dtype:
            raise ValueError("%s: the caches must have one shape and type" % name)
        s = t.stride()
        gap = 1
        for st, n in sorted(zip(s[lead + 1:], inside)):
            if n > 1:
                if st != gap:
                    raise ValueError("%s: a page must be one piece of memory" % name)
                gap *= n
        ptrs.append(t.data_ptr())
        layer.append(s[0] * size if lead and shape[0] > 1 else 0)
        page.append(s[lead] * size if shape[lead] > 1 else 0)
    _launch(first, "amp_b200_copy_pages", ptrs.buffer_info()[0], layer.buffer_info()[0], page.buffer_info()[0], len(caches),
            shape[0] if lead else 1, shape[lead], count * size, src.buffer_info()[0], dst.buffer_info()[0], len(src))
    return caches
