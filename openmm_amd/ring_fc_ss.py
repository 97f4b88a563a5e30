"""Products of secret shares with cleartext weights in Z_{2^l}, grouped by expert: the online half of an FC layer whose
ciphertext work ran ahead of the input.

``HomFCSS`` multiplies one encrypted vector with one matrix when the input arrives.  With the weights fixed, the client can
send Enc(r) for a random r beforehand (``HomFCSS.encryptInputVector``), the server computes Enc(W r - s) and keeps s
(``matVecMul``), the client decrypts W r - s, which will be its share of the result.  Online the client sends x0 - r in the
clear and the server, which holds x1, computes its share

    y1 = W (x0 - r + x1) + s  mod 2^l        (``RingFCSS.matMul``: x = x0 - r, share1 = x1, add = s)

so that y0 + y1 = W (x0 + x1).  ``PreparedFCSS`` is that layer for both parties; rows of several experts (adapters, clients'
models) go through one call, and which row belongs to which expert is public.  Same ``gemini::Code`` errors as the other layer
classes.

``PreparedFCSS`` knows the rows of each matrix when it prepares them, before there is an input, so it serves adapters and clients'
models; experts chosen by what a token holds need a protocol of their own around ``RingFCSS.matMul`` (``rows``), as do rings wider
than a BFV context's plain modulus (below every prime of the context, 60 bits at most: l <= 59, and 48 with primes of 60 and 49
bits).
"""
import ctypes as C
import functools

import torch

from . import lib as L


_INT64 = torch.int64
_stream_of, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _need(cond, code, what):
    if not cond:
        raise L.MMHError(code, what)


def _rows_of(t, what, cols, dev):
    """a 2-D int64 tensor on CUDA device ``dev`` with contiguous rows of ``cols`` words -> its row stride in words"""
    if t.dtype is not _INT64 or t.dim() != 2 or t.get_device() != dev:
        raise L.MMHError(7, f"{what}: expected a 2-D int64 tensor on the weights' device")
    n, c = t.shape
    step, one = t.stride()
    if c != cols:
        raise L.MMHError(3, f"{what}: {c} columns instead of {cols}")
    if one != 1 and c > 1 and n:
        raise L.MMHError(7, f"{what}: rows must be contiguous")
    return step if n > 1 else c


def _index(t, what, dev):
    if t.dtype is not _INT64 or t.dim() != 1 or t.get_device() != dev or not t.is_contiguous():
        raise L.MMHError(7, f"{what}: expected a contiguous 1-D int64 tensor on the weights' device")
    return t.shape[0]


class RingWeights:
    """Weights [groups, rows, cols] (or [rows, cols]) laid out once as byte digits (mmh_ring_weights_create).  ``w``: signed
    integers int8 / int16 / int32 / int64 on the GPU; congruent modulo 2^ring_bw is the same weight."""

    def __init__(self, w, ring_bw):
        self.handle = L._vp()
        self.lib = L.load_library()
        _need(isinstance(w, torch.Tensor) and w.is_cuda and w.dtype in (torch.int8, torch.int16, torch.int32, torch.int64), 7,
              "encodeWeights: expected an int8, int16, int32 or int64 CUDA tensor")
        _need(w.dim() in (2, 3), 3, "encodeWeights: weight shape")
        w = w.contiguous()
        self.device = w.get_device()
        self._words = {}
        g, rows, cols = w.shape if w.dim() == 3 else (1, *w.shape)
        with torch.cuda.device(w.device):
            L.check(self.lib.mmh_ring_weights_create(L.dptr(w), w.element_size(), g, rows, cols, ring_bw, L._stream_ptr(),
                                                     C.byref(self.handle)))
        d = L._int()
        L.check(self.lib.mmh_ring_weights_info(self.handle, None, None, None, None, C.byref(d)))
        self.groups, self.rows, self.cols, self.ring_bw, self.digits = g, rows, cols, ring_bw, d.value

    def workspace(self, n):
        """scratch words of a call of n rows"""
        words = self._words.get(n)
        if words is None:
            c = L._sz()
            L.check(self.lib.mmh_ring_matmul_workspace(self.handle, n, C.byref(c)))
            if len(self._words) >= 256:
                self._words.clear()
            words = self._words[n] = c.value
        return words

    def close(self):
        if self.handle:
            self.lib.mmh_ring_weights_destroy(self.handle)
            self.handle = L._vp()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class RingFCSS:
    """setUp(ring_bw), encodeWeights once per layer, matMul per call."""

    def __init__(self):
        self.ring_bw = None

    def setUp(self, ring_bw):
        _need(2 <= ring_bw <= 64, 7, "setUp: ring_bw")
        self.ring_bw = ring_bw
        return 0

    def encodeWeights(self, w):
        _need(self.ring_bw is not None, 1, "encodeWeights: setUp first")
        return RingWeights(w, self.ring_bw)

    def matMul(self, weights, x, offsets=None, rows=None, share1=None, add=None, out=None):
        """out[r] = add[r] + W_g (x[t] + share1[t]) mod 2^l for offsets[g] <= r < offsets[g + 1], t = rows[r].

        x, share1 [tokens, cols]; rows int64 [n] (None: row r reads token r); offsets int64 [groups + 1] on the device (None
        with one group); add [n, w.rows] or [w.rows]; out [n, w.rows] (a new tensor with zeros in rows of no group
        when None).  2-D operands may have any row stride of a row or more, and all but out a stride of 0.  add may be out;
        otherwise out shares no word with the other operands."""
        if self.ring_bw is None:
            raise L.MMHError(1, "matMul: setUp first")
        if not isinstance(weights, RingWeights) or not weights.handle or weights.ring_bw != self.ring_bw:
            raise L.MMHError(7, "matMul: weights")
        dev, cols, wide = weights.device, weights.cols, weights.rows
        ldx = _rows_of(x, "matMul: x", cols, dev)
        n = tokens = x.shape[0]
        px1 = ldx1 = prows = poff = padd = ldadd = pws = 0
        if share1 is not None:
            ldx1, px1 = _rows_of(share1, "matMul: share1", cols, dev), share1.data_ptr()
            _need(share1.shape[0] == tokens, 3, "matMul: #shares")
        if rows is not None:
            n, prows = _index(rows, "matMul: rows", dev), rows.data_ptr()
        if offsets is not None:
            _need(_index(offsets, "matMul: offsets", dev) == weights.groups + 1, 3, "matMul: offsets")
            poff = offsets.data_ptr()
        else:
            _need(weights.groups == 1, 2, "matMul: offsets")
        if add is not None:
            padd = add.data_ptr()
            if add.dim() == 1:
                _rows_of(add[None], "matMul: add", wide, dev)
            else:
                ldadd = _rows_of(add, "matMul: add", wide, dev)
                _need(add.shape[0] == n, 3, "matMul: add")
        new = out is None
        if new:
            out, ldo = x.new_empty((n, wide)), wide
        else:
            ldo = _rows_of(out, "matMul: out", wide, dev)
            _need(out.shape[0] == n, 3, "matMul: out")
        if n == 0:
            return out
        px = x.data_ptr()
        if not new:
            po = out.data_ptr()
            end = po + 8 * ((n - 1) * ldo + wide)
            operands = [(px, ldx, tokens, cols), (px1, ldx1, tokens, cols), (prows, 0, 1, n), (poff, 0, 1, weights.groups + 1)]
            if padd != po or (ldadd != ldo and n > 1):
                operands.append((padd, ldadd, n, wide))
            for p, ld, count, width in operands:
                if p < end and po < p + 8 * ((count - 1) * ld + width):
                    _need(not L.rows_overlap((po, wide, ((n, ldo),)), (p, width, ((count, ld),))), 7, "matMul: out overlaps an operand")
        words = weights.workspace(n)
        if words:
            ws = x.new_empty(words)
            pws = ws.data_ptr()
        rc = weights.lib.mmh_ring_matmul(weights.handle, px, ldx, px1, ldx1, tokens, prows, poff, n, padd, ldadd,
                                         out.data_ptr(), ldo, new, pws, words, _stream_of(dev))
        if rc:
            L.check(rc)
        return out


def _on_its_device(method):
    """HomFCSS and the samplers work on the current device's stream, so the layer makes its context's device the current one"""
    @functools.wraps(method)
    def call(self, *args, **kwargs):
        dev = None if self.sampler is None else self.ctx.device
        if dev is None or dev == (_current_device() if torch.cuda.is_initialized() else 0):
            return method(self, *args, **kwargs)
        with torch.cuda.device(dev):
            return method(self, *args, **kwargs)
    return call


class PreparedFCSS:
    """An FC layer of n rows over one or more weight matrices whose ciphertext work precedes the input.  BOB:

        cts = bob.prepareMasks(n, meta)          -> ALICE   (one Enc(r) per row)
        bob.finishMasks(out_cts)                 <- ALICE   (out_cts of prepareRows)
        opened, y0 = bob.openInput(x0)           -> ALICE   (x0 - r; y0 is BOB's share of the result)

    ALICE:  prepareWeights(w) once, out_cts = prepareRows(cts, offsets), y1 = online(opened, x1).

    Rows offsets[g] .. offsets[g + 1] use matrix g.  A mask serves one input: a second openInput, or online, needs new masks.
    setUp, new masks, new weights and new rows each drop what was prepared before them.
    The ciphertext work is per row: 2048 -> 1001 in the ring 2^37 about 0.05 ms for a mask, 0.1 to 0.2 ms for its product and
    0.03 ms to decrypt it, beside 0.05 ms online for 64 rows together.
    ``exact`` keeps the noise terms the approximate re-sharing of ``HomFCSS.matVecMul`` leaves out (shares then add up exactly,
    otherwise within 1)."""

    def __init__(self):
        from .hom_fc_ss import HomFCSS
        self.fc, self.ring = HomFCSS(), RingFCSS()
        self._forget()

    def _forget(self):
        self.sampler = self.weights = self._plain = self._masks = self._y0 = self._s = self._offsets = None

    def setUp(self, ctx, sampler, sk_ntt=None, pk_ntt=None, exact=False):
        _need(ctx.t >= 4 and ctx.t & (ctx.t - 1) == 0, 1, "setUp: the plain modulus is not a ring 2^l")
        of = lambda c: (c.N, c.q, c.device)
        _need(of(sampler.ctx) == of(ctx), 7, "setUp: the sampler draws for another context")
        self._forget()
        self.ctx, self.sampler, self.exact = ctx, sampler, exact
        self.fc.setUp(ctx, sk_ntt=sk_ntt, pk_ntt=pk_ntt)
        self.ring.setUp(ctx.t.bit_length() - 1)
        return 0

    # -- BOB
    @_on_its_device
    def prepareMasks(self, n, meta):
        _need(self.sampler is not None, 1, "prepareMasks: setUp first")
        self._masks = self._y0 = None
        cols, p = meta.input_shape[0], self.fc.plan(meta)
        r = (self.sampler.words(n * cols) & (self.ctx.t - 1)).view(n, cols)
        cts = [self.fc.encryptInputVector(v, meta, (self.sampler.uniform(p.n_in), self.sampler.noise(p.n_in))) for v in r]
        self._masks, self._mask_meta = r, meta
        return cts

    @_on_its_device
    def finishMasks(self, out_cts):
        _need(self._masks is not None and len(out_cts) == self._masks.shape[0], 3, "finishMasks: #rows")
        y0 = self._masks.new_empty((len(out_cts), self._mask_meta.weight_shape[0]))
        for row, ct in zip(y0, out_cts):
            row.copy_(self.fc.decryptToVector(ct, self._mask_meta))
        self._y0 = y0

    @_on_its_device
    def openInput(self, x0):
        _need(self._y0 is not None, 1, "openInput: no masks that were not used")
        _need(tuple(x0.shape) == tuple(self._masks.shape), 3, "openInput: input shape")
        opened, y0 = (x0 - self._masks) & (self.ctx.t - 1), self._y0
        self._masks = self._y0 = None
        return opened, y0

    # -- ALICE
    @_on_its_device
    def prepareWeights(self, w, meta):
        """w [groups, rows, cols], int8 to int64 ring elements (values below 2^l or signed)"""
        _need(self.sampler is not None, 1, "prepareWeights: setUp first")
        _need(w.dim() == 3 and tuple(w.shape[1:]) == tuple(meta.weight_shape), 3, "prepareWeights: weight shape")
        self.weights = self._plain = self._s = self._offsets = None
        weights, self._meta = self.ring.encodeWeights(w), meta
        self._plain = [self.fc.encodeWeightMatrix(m, meta) for m in (w.to(_INT64) & (self.ctx.t - 1)).contiguous()]
        self.weights = weights

    @_on_its_device
    def prepareRows(self, cts, offsets):
        """the ciphertexts of W_g r - s for BOB; offsets: groups + 1 integers on the host, every row in a group"""
        offsets = [int(v) for v in offsets]
        _need(self.weights is not None, 1, "prepareRows: prepareWeights first")
        _need(len(offsets) == self.weights.groups + 1 and offsets[0] == 0 and offsets[-1] == len(cts) and
              all(a <= b for a, b in zip(offsets, offsets[1:])), 3, "prepareRows: offsets")
        self._s = self._offsets = None
        from .hom_fc_ss import Meta
        meta = Meta(self._meta.weight_shape, self._meta.input_shape, False)    # the mask is BOB's alone
        n, N, smp, out, s = self.fc.plan(meta).n_out, self.ctx.N, self.sampler, [], []
        for g, plain in enumerate(self._plain):
            for ct in cts[offsets[g]:offsets[g + 1]]:
                if self.exact:
                    rand = (smp.words(n * N).view(n, N), smp.ternary(n), smp.noise(n), smp.noise(n), smp.words(n * N).view(n, N))
                else:
                    rand = smp.reshare(n)
                c, share = self.fc.matVecMul(plain, ct, None, meta, rand, exact=self.exact)
                out.append(c)
                s.append(share)
        dev = self.weights.device
        self._s = torch.stack(s) if s else torch.empty((0, self.weights.rows), dtype=_INT64, device=f"cuda:{dev}")
        self._offsets = torch.tensor(offsets, dtype=_INT64, device=f"cuda:{dev}")
        return out

    @_on_its_device
    def online(self, opened, share1):
        _need(self._s is not None, 1, "online: no rows prepared that were not used")
        _need(opened.shape[0] == self._s.shape[0], 3, "online: #rows")
        y1 = self.ring.matMul(self.weights, opened, self._offsets, share1=share1, add=self._s, out=self._s)
        self._s = self._offsets = None
        return y1
