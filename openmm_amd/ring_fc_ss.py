"""Products of secret shares with cleartext weights in Z_{2^l}, grouped by expert: the online half of an FC layer whose
ciphertext work ran ahead of the input.

``HomFCSS`` multiplies one encrypted vector with one matrix when the input arrives.  With the weights fixed, the client can
send Enc(r) for a random r beforehand (``HomFCSS.encryptInputVector``), the server computes Enc(W r - s) and keeps s
(``matVecMul``), the client decrypts W r - s, which will be its share of the result.  Online the client sends x0 - r in the
clear and the server, which holds x1, computes its share

    y1 = W (x0 - r + x1) + s  mod 2^l        (``RingFCSS.matMul``: x = x0 - r, share1 = x1, add = s)

so that y0 + y1 = W (x0 + x1).  Rows of several experts (adapters, clients' models) go through one call; which row belongs
to which expert is public.  Same ``gemini::Code`` errors as the other layer classes.
"""
import ctypes as C

from . import lib as L


def _need(cond, code, what):
    if not cond:
        raise L.MMHError(code, what)


def _rows_of(t, what, cols=None):
    """a 2-D int64 CUDA tensor with contiguous rows -> its row stride in words"""
    import torch
    _need(isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.int64 and t.dim() == 2, 7,
          f"{what}: expected a 2-D int64 CUDA tensor")
    _need(cols is None or t.shape[1] == cols, 3, f"{what}: {t.shape[1]} columns instead of {cols}")
    _need(t.shape[1] <= 1 or t.numel() == 0 or t.stride(1) == 1, 7, f"{what}: rows must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _index(t, what, device):
    import torch
    _need(isinstance(t, torch.Tensor) and t.dtype == torch.int64 and t.dim() == 1 and t.is_contiguous(), 7,
          f"{what}: expected a contiguous 1-D int64 tensor")
    _need(t.device == device, 7, f"{what}: on another device than the weights")
    return t


class RingWeights:
    """Weights [groups, rows, cols] (or [rows, cols]) laid out once as byte digits (mmh_ring_weights_create).  ``w``: signed
    integers int8 / int16 / int32 / int64 on the GPU; congruent modulo 2^ring_bw is the same weight."""

    def __init__(self, w, ring_bw):
        import torch
        self.handle = L._vp()
        self.lib = L.load_library()
        _need(isinstance(w, torch.Tensor) and w.is_cuda and w.dtype in (torch.int8, torch.int16, torch.int32, torch.int64), 7,
              "encodeWeights: expected an int8, int16, int32 or int64 CUDA tensor")
        _need(w.dim() in (2, 3), 3, "encodeWeights: weight shape")
        w = w.contiguous()
        self.device = w.device
        g, rows, cols = w.shape if w.dim() == 3 else (1, *w.shape)
        with torch.cuda.device(w.device):
            L.check(self.lib.mmh_ring_weights_create(L.dptr(w), w.element_size(), g, rows, cols, ring_bw, L._stream_ptr(),
                                                     C.byref(self.handle)))
        d = L._int()
        L.check(self.lib.mmh_ring_weights_info(self.handle, None, None, None, None, C.byref(d)))
        self.groups, self.rows, self.cols, self.ring_bw, self.digits = g, rows, cols, ring_bw, d.value

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
        with one group); add [n, w.rows] or [w.rows]; out [n, w.rows] (a new tensor of zeros behind the last group when
        None).  2-D operands may have any row stride.  add may be out."""
        import torch
        _need(self.ring_bw is not None, 1, "matMul: setUp first")
        _need(isinstance(weights, RingWeights) and bool(weights.handle) and weights.ring_bw == self.ring_bw, 7, "matMul: weights")
        ldx = _rows_of(x, "matMul: x", weights.cols)
        _need(x.device == weights.device, 7, "matMul: x on another device than the weights")
        tokens, ldx1 = x.shape[0], 0
        if share1 is not None:
            ldx1 = _rows_of(share1, "matMul: share1", weights.cols)
            _need(share1.shape[0] == tokens and share1.device == x.device, 3, "matMul: #shares")
        n = tokens if rows is None else _index(rows, "matMul: rows", x.device).numel()
        if offsets is None:
            _need(weights.groups == 1, 2, "matMul: offsets")
        else:
            _need(_index(offsets, "matMul: offsets", x.device).numel() == weights.groups + 1, 3, "matMul: offsets")
        ldadd = 0
        if add is not None:
            ldadd = _rows_of(add if add.dim() == 2 else add[None], "matMul: add", weights.rows)
            ldadd = ldadd if add.dim() == 2 else 0
            _need((add.dim() == 1 or add.shape[0] == n) and add.device == x.device, 3, "matMul: add")
        if out is None:
            # with offsets, rows behind the last group are not written
            new = torch.empty if offsets is None else torch.zeros
            out = new((n, weights.rows), dtype=torch.int64, device=x.device)
        ldo = _rows_of(out, "matMul: out", weights.rows)
        _need(out.shape[0] == n and out.device == x.device, 3, "matMul: out")
        ptr = lambda t: L._vp(0 if t is None else t.data_ptr())
        s = L._vp(torch.cuda.current_stream(x.device).cuda_stream)
        L.check(weights.lib.mmh_ring_matmul(weights.handle, ptr(x), ldx, ptr(share1), ldx1, tokens, ptr(rows), ptr(offsets), n,
                                            ptr(add), ldadd, ptr(out), ldo, s))
        return out
