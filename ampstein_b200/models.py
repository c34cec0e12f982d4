"""Host-side mirror of the reference's linear classes and CUDA-graph decode step, restricted to
the EXL3 linears (reference: src/ucode/ampstein/models.uc:49-107 LinearEXL3,
src/ucode/ampstein/graphdec.uc:151-282 step capture and replay), and a paged key-value cache with
the attention block over it.

LinearEXL3 derives everything from the trellis tensor:
    K = trellis.shape[-1] / 16, in_features = trellis.shape[0] * 16, out_features = shape[1] * 16
forward(x) picks the many-rows operator above RECON_ROWS rows, the decode operator otherwise,
exactly as the reference does.
"""
import torch

from . import attention, exl3

RECON_ROWS = 144          # models.uc:36
RECON_MAX_N = 32768       # models.uc:37


class LinearEXL3:
    def __init__(self, trellis, suh, svh, bias=None, mul1=False, mcg=False):
        if mul1 and mcg:
            raise ValueError("LinearEXL3: both mul1 and mcg set")
        if trellis.dim() != 3 or trellis.shape[2] % 8:
            raise ValueError("LinearEXL3: trellis must be (k/16, n/16, 16 K)")
        if trellis.shape[2] % 16 and not (mul1 and 1 <= trellis.shape[2] // 16 <= 3):
            # (reference: models.uc:9-15, 68-71: K = shape[2] / 16 as a float; bits_k.cuh:14-20)
            raise ValueError("LinearEXL3: half-integer bitrates are 1.5 / 2.5 / 3.5 with the mul1 codebook")
        self.trellis, self.suh, self.svh, self.bias = trellis, suh, svh, bias
        self.K = trellis.shape[2] // 16 if trellis.shape[2] % 16 == 0 else trellis.shape[2] / 16.0     # 1.5 / 2.5 / 3.5: 16 K + 8 words
        self.mul1, self.mcg = mul1, mcg
        self.in_features = trellis.shape[0] * 16
        self.out_features = trellis.shape[1] * 16
        self._plan = None

    def _biased(self, y, out):
        """y, the product, and the bias; in `out` where the caller gave it"""
        if self.bias is None:
            return y
        return y.add(self.bias) if out is None else y.add_(self.bias)

    def forward(self, x, out=None):
        m = x.shape[0]
        if out is None and m <= RECON_ROWS:
            # the per-token call: the weight is checked in full when it is not what it was
            plan = self._plan
            if plan is None or not plan.matches(self.trellis, self.suh, self.svh, self.mul1, self.mcg):
                plan = self._plan = exl3.GemmPlan(self.trellis, self.suh, self.svh, self.mul1, self.mcg)
            y = plan.run(x, self.trellis, self.suh, self.svh)
            if y is not None:
                return y if self.bias is None else y.add(self.bias)
        if out is None and m > RECON_ROWS and self.out_features <= RECON_MAX_N:
            y = exl3.exl3_gemm_recon(x.contiguous(), self.trellis, self.suh, self.svh, self.K,
                                     self.mul1, self.mcg)
        else:
            y = x.new_empty((m, self.out_features), dtype=torch.float16) if out is None else out
            exl3.exl3_gemm(x, self.trellis, y, self.suh, self.svh, self.mul1, self.mcg)
        return self._biased(y, out)

    def forward_silu_mul(self, gate, up, out=None):
        """out = this linear of silu(gate) * up in one launch (the down projection behind a gate|up
        bundle, up to 16 rows); larger batches take the two-step path of the caller."""
        m = gate.shape[0]
        y = torch.empty((m, self.out_features), dtype=torch.float16, device=gate.device) if out is None else out
        exl3.exl3_gemm_silu_mul(gate, up, self.trellis, y, self.suh, self.svh, self.mul1, self.mcg)
        return self._biased(y, out)

    def forward_add_res(self, x, h, y, ssq):
        """y = fp16(h + this linear of x), ssq = block sums of squares of y: the linear and the residual
        add of the norm that follows, in one launch (up to 16 rows). Not for linears with a bias, which the launch does not add."""
        if self.bias is not None:
            raise ValueError("LinearEXL3.forward_add_res: the linear has a bias")
        return exl3.exl3_gemm_add_res(x, self.trellis, self.suh, self.svh, h, y, ssq, self.mul1, self.mcg)

    def weight_bytes(self):
        return self.trellis.numel() * 2


def linear(ws, key, dev=0):
    """EXL3 linear `key` of a weight set on device `dev` (reference: models.uc LinearEXL3(ws, key, dev),
    :49-110): <key>.trellis / .suh / .svh (+ optional .bias), the codebook from the marker tensors
    <key>.mul1 / <key>.mcg (mutually exclusive), the bitrate from the trellis shape."""
    mul1, mcg = ws.has(key + ".mul1"), ws.has(key + ".mcg")
    if mul1 and mcg:
        raise ValueError("LinearEXL3: %s: both .mul1 and .mcg marker tensors present" % key)
    bias = ws.gpu16(key + ".bias", dev) if ws.has(key + ".bias") else None
    return LinearEXL3(ws.gpu(key + ".trellis", dev), ws.gpu(key + ".suh", dev), ws.gpu(key + ".svh", dev), bias=bias,
                      mul1=mul1, mcg=mcg)


def split_n(total, unit, weights):
    """Cut `total` (a multiple of `unit`) into per-rank [start, length] ranges proportional to
    `weights` by largest remainder (reference: src/ucode/ampstein/qwen35_tp.uc:40-72)."""
    n, tot = total // unit, float(sum(weights))
    cnt, rem, used = [], [], 0
    for g, w in enumerate(weights):
        exact = n * w / tot
        c = int(exact)
        cnt.append(c)
        rem.append((exact - c, g))
        used += c
    rem.sort(key=lambda a: (-a[0], a[1]))
    k = 0
    while used < n:
        cnt[rem[k % len(weights)][1]] += 1
        k += 1
        used += 1
    out, at = [], 0
    for c in cnt:
        out.append((at * unit, c * unit))
        at += c
    return out


def cols(lin, ranges):
    """Column-parallel shard: output columns ([start, length] pairs, 256-aligned) concatenated;
    suh whole, svh and the bias sliced (reference: models.uc cols(), :537-545)."""
    for n0, w in ranges:
        if n0 % 128 or w % 128 or n0 < 0 or w <= 0 or n0 + w > lin.out_features:
            raise ValueError("models.sub_columns: range [%d, %d] not 128-aligned/in bounds" % (n0, w))
    if lin.trellis.is_cuda:
        tr, svh = exl3.exl3_shard_cols(lin.trellis, lin.svh, ranges)        # one launch on the device
    else:
        # weights still in host memory (before the upload): plain slices of the host tensors
        tr = torch.cat([lin.trellis[:, n0 // 16:(n0 + w) // 16] for n0, w in ranges], dim=1).contiguous()
        svh = torch.cat([lin.svh[n0:n0 + w] for n0, w in ranges]).contiguous()
    bias = None if lin.bias is None else torch.cat([lin.bias[n0:n0 + w] for n0, w in ranges])
    return LinearEXL3(tr, lin.suh, svh, bias=bias, mul1=lin.mul1, mcg=lin.mcg)


def rows(lin, k0, klen):
    """Row-parallel shard: input rows [k0, k0 + klen), 128-aligned, with the matching suh slice
    and the whole svh; the shards' outputs SUM to the full product (reference: models.uc rows(),
    :547-562). The shard of the first rows has the bias."""
    if k0 % 128 or klen % 128 or k0 < 0 or klen <= 0 or k0 + klen > lin.in_features:
        raise ValueError("models.rows: range [%d, %d] not 128-aligned/in bounds" % (k0, klen))
    if lin.trellis.is_cuda:
        tr, suh = exl3.exl3_shard_rows(lin.trellis, lin.suh, k0, klen)
    else:
        tr, suh = lin.trellis[k0 // 16:(k0 + klen) // 16].clone(), lin.suh[k0:k0 + klen].clone()
    return LinearEXL3(tr, suh, lin.svh, bias=lin.bias if k0 == 0 else None, mul1=lin.mul1, mcg=lin.mcg)


def _bundle_check(linears):
    a = linears[0]
    for i, w in enumerate(linears[1:], 1):
        if (w.K, w.mul1, w.mcg, w.in_features) != (a.K, a.mul1, a.mcg, a.in_features):
            raise ValueError("models.bundle: fused linears must share K, in_features and codebook "
                             "(matrix %d differs)" % i)


def _add_biases(linears, outs):
    """What LinearEXL3.forward does behind the product, for the outputs of a bundle; in place"""
    for i, w in enumerate(linears):
        if w.bias is not None:
            outs[i].add_(w.bias)


def _first_rows(t, m):
    """The beginning of a (num, rows, n) buffer as (num, m, n)"""
    return t if m == t.shape[1] else t.view(-1)[:t.shape[0] * m * t.shape[2]].view(t.shape[0], m, t.shape[2])


def _bundle_rows(x, most):
    m = x.shape[1]
    if not 1 <= m <= most:
        raise ValueError("models.bundle: %d rows, the bundle's buffers hold %d" % (m, most))
    return m


class Multi:
    """Equal-shape bundle (reference: models.uc multi(), :338-361): run(x) writes all outputs
    stacked into `out` (num, m, n) with ONE launch, and one more for each linear with a bias. x is (1, m, k);
    with fewer rows than `out` has, the outputs are stacked at its beginning. Returns them, (num, rows of x, n)."""

    def __init__(self, linears, out):
        _bundle_check(linears)
        dev = out.device
        self.linears, self.out = linears, out
        self.B = exl3.ptr_array([w.trellis.data_ptr() for w in linears], dev)
        self.suh = exl3.ptr_array([w.suh.data_ptr() for w in linears], dev)
        self.svh = exl3.ptr_array([w.svh.data_ptr() for w in linears], dev)

    def run(self, x, a_had=None):
        """a_had: (num, m, k) fp16 scratch, used from five rows up (allocated here if missing)"""
        a = self.linears[0]
        m = _bundle_rows(x, self.out.shape[1])
        out = _first_rows(self.out, m)
        if a_had is None and (m >= 5 or x.dtype == torch.bfloat16):
            a_had = torch.empty((len(self.linears), m, a.in_features), dtype=torch.float16, device=x.device)
        exl3.mgemm(x, self.B, out, self.suh, a_had, self.svh, a.K, a.mcg, a.mul1)
        _add_biases(self.linears, out)
        return out

    def run_norm(self, x, res, norm_w, eps, y):
        """The bundle applied to RMSNorm(x + res) * norm_w, y = fp16(x + res): one launch (up to 16 rows)."""
        out = _first_rows(self.out, _bundle_rows(x, self.out.shape[1]))
        _run_norm(self, out, x, res, norm_w, eps, y, None)
        _add_biases(self.linears, out)
        return out

    def run_normed(self, y, ssq, norm_w, eps):
        """The bundle applied to the norm of a residual stream whose block sums of squares the producing
        linear left in ssq (LinearEXL3.forward_add_res)."""
        a = self.linears[0]
        out = _first_rows(self.out, _bundle_rows(y, self.out.shape[1]))
        exl3.mgemm_normed(y, ssq, norm_w, eps, self.B, out, self.suh, self.svh, a.K, a.mcg, a.mul1)
        _add_biases(self.linears, out)
        return out


def _run_norm(bundle, carrier, x, res, norm_w, eps, y, opts):
    a = bundle.linears[0]
    return exl3.mgemm_rms_norm_res(x, res, norm_w, eps, y, bundle.B, carrier, bundle.suh, bundle.svh, a.K, a.mcg, a.mul1, opts)


class Sliced:
    """Bundle for unequal widths such as Q/K/V (reference: models.uc sliced(), :367-432): every
    matrix is cut into column slices of the widths' gcd (a multiple of 128); outputs are written
    in place into `outs`, one (1, m, out_features) buffer per linear; biases are added there, a launch each.
    An x of fewer rows than the buffers have goes into their first rows. Returns the outputs of x's rows."""

    def __init__(self, linears, outs):
        import math
        _bundle_check(linears)
        dev = outs[0].device
        width = 0
        for w in linears:
            width = math.gcd(width, w.out_features)
        if width % 128 or width < 128:
            raise ValueError("models.sliced: unsuitable slice width %d" % width)
        t, svh, cp, stride, src = [], [], [], [], []
        for i, w in enumerate(linears):
            tw = w.trellis.shape[2]
            for n0 in range(0, w.out_features, width):
                t.append(w.trellis.data_ptr() + (n0 // 16) * tw * 2)
                svh.append(w.svh.data_ptr() + n0 * 2)
                cp.append(outs[i].data_ptr() + n0 * 2)
                stride.append(w.out_features)
                src.append(i)
        self.linears, self.outs, self.width, self.slices = linears, outs, width, len(t)
        m = outs[0].shape[1]
        self.B = exl3.ptr_array(t, dev)
        self.svh = exl3.ptr_array(svh, dev)
        self.suh = exl3.ptr_array([w.suh.data_ptr() for w in linears], dev)
        i32 = dict(dtype=torch.int32, device=dev)
        self.opts = {
            "size_n_list": torch.tensor([width] * len(t), **i32),
            "c_ptrs": exl3.ptr_array(cp, dev),
            "n_stride_list": torch.tensor(stride, **i32),
            "had_src_list": torch.tensor(src, **i32),
            "num_had_src": len(linears),
        }
        # descriptor only: (num_slices, m, width); the data goes through c_ptrs
        self.carrier = torch.empty((len(t), m, width), dtype=torch.float16, device=dev)

    def _rows(self, x):
        """The descriptor and the buffers for x's rows"""
        m = _bundle_rows(x, self.carrier.shape[1])
        if m == self.carrier.shape[1]:
            return self.carrier, self.outs
        return _first_rows(self.carrier, m), [t[:, :m] for t in self.outs]

    def run(self, x, a_had=None):
        """a_had: (linears, m, k) fp16 scratch, used from five rows up (allocated here if missing)"""
        a = self.linears[0]
        m = x.shape[1]
        carrier, outs = self._rows(x)
        if a_had is None and (m >= 5 or x.dtype == torch.bfloat16):
            a_had = torch.empty((len(self.linears), m, a.in_features), dtype=torch.float16, device=x.device)
        exl3.mgemm(x, self.B, carrier, self.suh, a_had, self.svh, a.K, a.mcg, a.mul1, self.opts)
        _add_biases(self.linears, outs)
        return outs

    def run_norm(self, x, res, norm_w, eps, y):
        """The bundle applied to RMSNorm(x + res) * norm_w, y = fp16(x + res): one launch (up to 16 rows)."""
        carrier, outs = self._rows(x)
        _run_norm(self, carrier, x, res, norm_w, eps, y, self.opts)
        _add_biases(self.linears, outs)
        return outs

    def run_normed(self, y, ssq, norm_w, eps):
        """The bundle applied to the norm of a residual stream whose block sums of squares the producing
        linear left in ssq (LinearEXL3.forward_add_res)."""
        a = self.linears[0]
        carrier, outs = self._rows(y)
        exl3.mgemm_normed(y, ssq, norm_w, eps, self.B, carrier, self.suh, self.svh, a.K, a.mcg, a.mul1, self.opts)
        _add_biases(self.linears, outs)
        return outs


class PagedCache:
    """Key-value cache of a model in pages: k, v (layers, pages, page_size, kv_heads, dim) and table (slots, max_pages) int32 on the
    device, the bookkeeping on the host. A sequence has a slot, that is a row of the table; its pages are the same in every layer.
    Forks share pages until one of them writes. Entries of pages that a sequence does not have (any more) are -1.

    The host knows every length (extend() announces tokens before they are written), nothing is read back. Calls that copy pages or
    change the table run on the current stream and do not wait: those of one cache belong on one stream, in the order of the work on it,
    and not inside a captured graph."""

    def __init__(self, layers, pages, page_size, kv_heads, dim, slots, max_pages, dtype=torch.float16, device="cuda"):
        if min(layers, pages, page_size, kv_heads, dim, slots, max_pages) < 1:
            raise ValueError("PagedCache: sizes must be positive")
        # (zeros: whatever a page holds behind a sequence's end is finite)
        self.k = torch.zeros((layers, pages, page_size, kv_heads, dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.table = torch.full((slots, max_pages), -1, dtype=torch.int32, device=device)
        self.page_size, self.max_pages = page_size, max_pages
        self._free = list(range(pages - 1, -1, -1))          # (popped from the end: low numbers first)
        self._uses = [0] * pages                              # sequences that have the page
        # per slot: [pages (None: given up), tokens, first position of the last extend(), first position that sees no given-up page]
        self._seqs = [None] * slots

    @property
    def free_pages(self):
        return len(self._free)

    def _seq(self, slot):
        if not 0 <= slot < len(self._seqs) or self._seqs[slot] is None:
            raise ValueError("PagedCache: slot %s holds no sequence" % (slot,))
        return self._seqs[slot]

    def length(self, slot):
        """Tokens announced for the sequence: the position of its next one"""
        return self._seq(slot)[1]

    def _write_row(self, slot):
        pages = self._seqs[slot][0] if self._seqs[slot] is not None else []
        row = [-1 if p is None else p for p in pages] + [-1] * (self.max_pages - len(pages))
        row = torch.tensor(row, dtype=torch.int32)
        if self.table.is_cuda:
            row = row.pin_memory()                           # (torch keeps the pinned memory until the copy is done: no wait here)
        self.table[slot].copy_(row, non_blocking=True)

    def _drop(self, page):
        self._uses[page] -= 1
        if self._uses[page] == 0:
            self._free.append(page)

    def add(self):
        """A slot for a new sequence"""
        for slot, seq in enumerate(self._seqs):
            if seq is None:
                self._seqs[slot] = [[], 0, 0, 0]
                return slot
        raise RuntimeError("PagedCache: all %d slots are taken" % len(self._seqs))

    def extend(self, slot, tokens):
        """Room for `tokens` more tokens of the sequence, which may then be written (rope_append). A page that a fork shares gets a
        copy of its own where they go into it. Returns the position of the first of them. RuntimeError, and nothing changed, without
        room."""
        seq = self._seq(slot)
        pages, at = seq[:2]
        if tokens < 0:
            raise ValueError("PagedCache.extend: tokens must not be negative")
        need = -(-(at + tokens) // self.page_size)
        if need > self.max_pages:
            raise RuntimeError("PagedCache: %d tokens do not fit into %d pages" % (at + tokens, self.max_pages))
        last = at // self.page_size if tokens and at % self.page_size else None           # the half-filled page that is written on
        own = last is not None and self._uses[pages[last]] > 1
        if need - len(pages) + own > len(self._free):
            raise RuntimeError("PagedCache: %d pages are free, %d are needed" % (len(self._free), need - len(pages) + own))
        changed = own
        if own:
            page = self._free[-1]
            attention.copy_pages([self.k, self.v], [pages[last]], [page])         # (may raise: nothing has changed yet)
            self._free.pop()
            self._drop(pages[last])
            self._uses[page] = 1
            pages[last] = page
        while len(pages) < need:
            page = self._free.pop()
            self._uses[page] = 1
            pages.append(page)
            changed = True
        seq[1] = at + tokens
        if tokens:
            seq[2] = at
        if changed:
            self._write_row(slot)
        return at

    def fork(self, slot):
        """A new sequence with the same tokens; shares the pages. Returns its slot."""
        pages, *rest = self._seq(slot)
        new = self.add()
        self._seqs[new] = [list(pages), *rest]
        for page in pages:
            if page is not None:
                self._uses[page] += 1
        self._write_row(new)
        return new

    def truncate(self, slot, tokens):
        """Takes back what stands behind the first `tokens` tokens (rejected drafts). ValueError, and nothing changed, where the next token
        would see a page that has been given up."""
        seq = self._seq(slot)
        if not 0 <= tokens <= seq[1]:
            raise ValueError("PagedCache.truncate: %d of %d tokens" % (tokens, seq[1]))
        keep = -(-tokens // self.page_size)
        gaps = None in seq[0][:keep]
        if gaps and tokens < seq[3]:
            raise ValueError("PagedCache.truncate: the token at position %d sees pages that have been given up (from %d on it does not)" % (tokens, seq[3]))
        for page in seq[0][keep:]:
            if page is not None:
                self._drop(page)
        changed = len(seq[0]) > keep
        del seq[0][keep:]
        seq[1:] = tokens, min(seq[2], tokens), seq[3] if gaps else 0
        if changed:
            self._write_row(slot)

    def leave_behind(self, slot, window, sinks=0, pending=None):
        """Gives up the pages that no further token of the sequence sees: those that hold neither one of the first `sinks` tokens nor one
        that is visible, in a window of so many tokens, from the first token still to run. pending: how many of the announced tokens have
        not run yet, or may be taken back (drafts). By default those of the last extend(), whose pages are then safe before and after they
        run; but of a sequence's first tokens, its prompt, the last one alone: a prompt runs first, or pending says how long it is."""
        seq = self._seq(slot)
        pages, at, last = seq[:3]
        if window < 1 or sinks < 0:
            raise ValueError("PagedCache.leave_behind: window must be positive, sinks not negative")
        if pending is None:
            pending = at - last if last else min(1, at)
        if not 0 <= pending <= at:
            raise ValueError("PagedCache.leave_behind: %s of %d tokens are pending" % (pending, at))
        changed = False
        for i in range(-(-sinks // self.page_size), max(0, at - pending - window + 1) // self.page_size):
            if pages[i] is not None:
                self._drop(pages[i])
                pages[i] = None
                seq[3] = max(seq[3], (i + 1) * self.page_size + window - 1)
                changed = True
        if changed:
            self._write_row(slot)

    def free(self, slot):
        """The sequence is over: its slot and the pages that no fork has are free again"""
        for page in self._seq(slot)[0]:
            if page is not None:
                self._drop(page)
        self._seqs[slot] = None
        self._write_row(slot)

    def compact(self):
        """Moves pages so that the used ones are the first of the pool (which may then be cut off, or given to another cache). Returns how
        many are used."""
        used = sum(1 for n in self._uses if n)
        src = [p for p in range(used, len(self._uses)) if self._uses[p]]
        dst = [p for p in range(used) if not self._uses[p]]
        if src:
            attention.copy_pages([self.k, self.v], src, dst)
            to = dict(zip(src, dst))
            for a, b in to.items():
                self._uses[b], self._uses[a] = self._uses[a], 0
            for slot, seq in enumerate(self._seqs):
                if seq is not None and any(p in to for p in seq[0]):
                    seq[0] = [to.get(p, p) for p in seq[0]]
                    self._write_row(slot)
        self._free = list(range(len(self._uses) - 1, used - 1, -1))
        return used


class PagedAttention:
    """The attention block of a decoder layer over a PagedCache: q|k|v bundle, rotary positions with the write into the cache,
    attention, o. One object serves prompts, drafted and single tokens, eagerly or inside a DecodeGraph, up to the rows that the
    bundle's buffers hold in a call (a longer prompt goes in chunks)."""

    def __init__(self, qkv, o, cache, layer, dim, inv_freq, mscale=1.0, interleaved=False, window=0, sinks=0, scale=None):
        widths = [w.out_features for w in qkv.linears]
        kv_heads = cache.k.shape[3]
        if len(widths) != 3 or cache.k.shape[4] != dim or widths[1] != kv_heads * dim or widths[2] != kv_heads * dim or widths[0] % (kv_heads * dim):
            raise ValueError("PagedAttention: q|k|v of %s columns do not fit a cache of %d heads of %d" % (widths, kv_heads, dim))
        if dim not in attention.WIDTHS:
            raise ValueError("PagedAttention: heads of %d values (the attention takes %s)" % (dim, ", ".join(map(str, attention.WIDTHS))))
        if o.in_features != widths[0]:
            raise ValueError("PagedAttention: o takes %d columns, q gives %d" % (o.in_features, widths[0]))
        if not 0 <= layer < cache.k.shape[0]:
            raise ValueError("PagedAttention: layer %d of %d" % (layer, cache.k.shape[0]))
        self.qkv, self.o, self.dim = qkv, o, dim
        self.k, self.v = cache.k[layer], cache.v[layer]
        self.rope = dict(interleaved=interleaved, mscale=mscale)
        self.inv_freq, self.view = inv_freq, dict(window=window, sinks=sinks, scale=scale)

    def run(self, x, pos, table, cu=None, out=None):
        """x (1, rows, hidden); pos, cu as paged_attention, table (seqs, max_pages) the sequences' rows of the cache's. Returns (rows,
        hidden)."""
        q, k, v = (t[0].view(t.shape[1], -1, self.dim) for t in self.qkv.run(x))
        q = attention.rope_append(q, k, v, pos, self.inv_freq, self.k, self.v, table, cu=cu, out=q, **self.rope)
        a = attention.paged_attention(q, self.k, self.v, table, pos, cu=cu, **self.view)
        return self.o.forward(a.view(a.shape[0], -1), out)


class DecodeGraph:
    """Captures `step_fn()` (a sequence of operator calls on fixed buffers) in one CUDA graph
    after warm-up runs, then replays it: one host->device crossing per step, as the reference's
    graphdec does. Everything the step touches must exist before capture."""

    def __init__(self, step_fn, warmup=3, stream=None):
        self.stream = stream if stream is not None else torch.cuda.Stream()
        with torch.cuda.stream(self.stream):
            for _ in range(warmup):
                step_fn()
            self.stream.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph, stream=self.stream):
                step_fn()
        torch.cuda.synchronize()

    def replay(self):
        self.graph.replay()
