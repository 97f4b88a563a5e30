"""Host-side mirror of ``gemini::HomConv2DSS`` (include/gemini/cheetah/hom_conv2d_ss.h:27-115).

Same method names, argument meaning and error codes as the reference class; ciphertexts and
plaintexts are device tensors ([n,2,limbs,N] / [n,N] int64 holding uint64 bits) instead of
``seal::Ciphertext`` / ``seal::Plaintext`` vectors, and the per-ciphertext thread-pool loops
are single batched calls into libmm_hip.  Randomness is passed in explicitly (``rand``) so a
caller -- or a parity test -- controls every sampled polynomial.
"""
import ctypes as C
from dataclasses import dataclass

from . import lib as L

VALID, SAME = 0, 1  # gemini::Padding (tensor_shape.h:11)


def torch_empty_flag(like):
    import torch
    return torch.empty(1, dtype=torch.int32, device=like.device)


def _mod_t(x, t):
    """int64 tensor holding uint64 bits, reduced mod t (power of two: mask; else torch remainder on
    the non-negative representatives the callers pass)"""
    return x & (t - 1) if t & (t - 1) == 0 else x % t


class ConvMetaC(C.Structure):
    _fields_ = [("in_c", C.c_int64), ("in_h", C.c_int64), ("in_w", C.c_int64), ("f_h", C.c_int64),
                ("f_w", C.c_int64), ("n_filters", C.c_int64), ("padding_same", C.c_int32),
                ("stride", C.c_int32), ("is_shared_input", C.c_int32)]


class ConvWorkC(C.Structure):
    """mmh_conv_work (include/mm_hip.h)"""
    _fields_ = [("direct_fresh", C.c_int32), ("direct_prepared", C.c_int32), ("taps", C.c_int64),
                ("taps_padded", C.c_int64), ("live_columns", C.c_int64 * 2), ("n_in", C.c_int64), ("n_out", C.c_int64),
                ("n_cslices", C.c_int64), ("n_spatial", C.c_int64), ("n_targets", C.c_int64), ("limbs", C.c_int64),
                ("poly_degree", C.c_int64)]


@dataclass
class Meta:
    """HomConv2DSS::Meta (hom_conv2d_ss.h:31-38)"""
    ishape: tuple            # (C, H, W)
    fshape: tuple            # (C, fh, fw)
    n_filters: int
    padding: int = VALID
    stride: int = 1
    is_shared_input: bool = True


class Plan:
    """geometry of one layer on the device (mmh_conv_plan)"""

    def __init__(self, ctx, meta):
        self.ctx, self.meta = ctx, meta
        if len(meta.ishape) != 3 or len(meta.fshape) != 3 or meta.ishape[0] != meta.fshape[0]:
            raise L.MMHError(7, "Conv2D: channels mismatch")
        m = ConvMetaC(meta.ishape[0], meta.ishape[1], meta.ishape[2], meta.fshape[1], meta.fshape[2],
                      meta.n_filters, int(meta.padding), int(meta.stride), int(meta.is_shared_input))
        self.handle = L._vp()
        L.check(ctx.lib.mmh_conv_plan_create(ctx.handle, C.byref(m), C.byref(self.handle)))
        a, b, c, d = L._sz(), L._sz(), L._sz(), L._sz()
        oshape, strides = (C.c_int64 * 3)(), (C.c_int64 * 3)()
        L.check(ctx.lib.mmh_conv_plan_info(self.handle, C.byref(a), C.byref(b), C.byref(c), C.byref(d), oshape,
                                           strides))
        self.n_in, self.n_cslices, self.n_spatial, self.n_out = a.value, b.value, c.value, d.value
        self.out_shape = tuple(int(x) for x in oshape)
        self.slice_strides = tuple(int(x) for x in strides)

    def work(self):
        """what one server call of this layer does (mmh_conv_plan_work): route, taps, live columns, counts"""
        w = ConvWorkC()
        L.check(self.ctx.lib.mmh_conv_plan_work(self.handle, C.byref(w)))
        return w

    def __del__(self):
        try:
            if self.handle:
                self.ctx.lib.mmh_conv_plan_destroy(self.handle)
                self.handle = L._vp()
        except Exception:
            pass


class PreparedFilters:
    """Static filters of one layer kept on the device in the form the server call consumes
    (mmh_conv_filters).  Not in the reference, which re-encodes per call."""

    def __init__(self, plan, filters, nonzero):
        self.plan, self.nonzero = plan, nonzero
        self.handle = L._vp()
        L.check(plan.ctx.lib.mmh_conv_filters_prepare(plan.handle, L.dptr(filters.contiguous()),
                                                      C.byref(self.handle), L._stream_ptr()))

    def __del__(self):
        try:
            if self.handle:
                self.plan.ctx.lib.mmh_conv_filters_destroy(self.handle)
                self.handle = L._vp()
        except Exception:
            pass


class HomConv2DSS:
    def __init__(self):
        self.ctx = self.sk_ntt = self.pk_ntt = None
        self._plans = {}
        self._verdicts = None   # page-locked verdict words + events, made on first use
        self._pending = []      # slots of calls made with defer_verdict, read by raise_pending()

    # HomConv2DSS::setUp (hom_conv2d_ss.cc:467-495): sk_ntt [L,N] (client), pk_ntt [2,L,N] (server)
    def setUp(self, ctx, sk_ntt=None, pk_ntt=None):
        if ctx is not self.ctx:
            self._plans = {}   # a plan holds its context's degree and limbs
        self.ctx, self.sk_ntt, self.pk_ntt = ctx, sk_ntt, pk_ntt
        self.pk_last = None if pk_ntt is None else pk_ntt[:, :1].contiguous()
        self.sk_last = None if sk_ntt is None else sk_ntt[:1].contiguous()
        return 0

    def plan(self, meta):
        key = (tuple(meta.ishape), tuple(meta.fshape), meta.n_filters, meta.padding, meta.stride,
               meta.is_shared_input)
        if key not in self._plans:
            self._plans[key] = Plan(self.ctx, meta)
        return self._plans[key]

    def _need(self, cond, code, what):
        if not cond:
            raise L.MMHError(code, what)

    def _check_rand(self, p, rand, names):
        """every sampled polynomial batch is [n_out, N]: the kernels index them with the plan's sizes"""
        self._need(len(rand) == len(names), 7, "conv2DSS: rand = (" + ", ".join(names) + ")")
        for r, name in zip(rand, names):
            self._need(r is not None and tuple(r.shape) == (p.n_out, self.ctx.N), 3, f"conv2DSS: {name} shape")

    # encryptImage (hom_conv2d_ss.cc:497-522); rand = (a [n_in,L,N] uniform, e [n_in,N] signed)
    def encryptImage(self, img, meta, rand):
        self._need(self.ctx is not None and self.sk_ntt is not None, 1, "encryptImage: no secret key")
        self._need(tuple(img.shape) == tuple(meta.ishape), 3, "encryptImage: image shape")
        p = self.plan(meta)
        a, e = rand
        out = self.ctx._empty(p.n_in, 2, self.ctx.L, self.ctx.N)
        L.check(self.ctx.lib.mmh_conv_encrypt_image(p.handle, L.dptr(self.sk_ntt), L.dptr(img), L.dptr(a),
                                                    L.dptr(e), L.dptr(out), L._stream_ptr()))
        return out

    # encodeImage (hom_conv2d_ss.cc:524-535)
    def encodeImage(self, img, meta):
        self._need(self.ctx is not None, 1, "encodeImage: no context")
        self._need(tuple(img.shape) == tuple(meta.ishape), 3, "encodeImage: image shape")
        p = self.plan(meta)
        out = self.ctx._empty(p.n_in, self.ctx.N)
        L.check(self.ctx.lib.mmh_conv_encode_image(p.handle, L.dptr(img), L.dptr(out), L._stream_ptr()))
        return out

    # encodeFilters (hom_conv2d_ss.cc:537-561): filters [M, C, fh, fw] -> [M, n_cslices, N]
    def encodeFilters(self, filters, meta):
        self._need(filters.shape[0] > 0 and filters.shape[0] == meta.n_filters, 7, "encodeFilters: #filters")
        self._need(tuple(filters.shape[1:]) == tuple(meta.fshape), 3, "encodeFilters: filter shape")
        p = self.plan(meta)
        out = self.ctx._empty(meta.n_filters, p.n_cslices, self.ctx.N)
        L.check(self.ctx.lib.mmh_conv_encode_filters(p.handle, L.dptr(filters), L.dptr(out), L._stream_ptr()))
        # a filter encodes to all-zero polynomials iff all its weights are 0 mod t: settle the
        # conv2DOneFilter :573-580 check here, on the small tensor, and remember the verdict
        out._mm_nonzero = L.DeferredFlag((_mod_t(filters, self.ctx.t) != 0).reshape(meta.n_filters, -1).any(dim=1).all())
        return out

    # conv2DSS (hom_conv2d_ss.cc:621-712); rand = (u [n_out,N], e1 [n_out,N], mask [n_out,N]) for the
    # shipped USE_APPROX_RESHARE build, (flood, u, e0, e1, mask) with exact=True for the other build
    def conv2DSS(self, img_share0, img_share1, filters, meta, rand, exact=False):
        self._need(self.pk_ntt is not None, 1, "conv2DSS: no public key")
        p = self.plan(meta)
        self._need(filters.shape[0] == meta.n_filters, 3, "conv2DSS: #filters")
        self._need(tuple(img_share0.shape) == (p.n_in, 2, self.ctx.L, self.ctx.N), 3, "conv2DSS: #ciphertexts")
        if meta.is_shared_input:
            self._need(img_share1 is not None and img_share1.shape[0] == img_share0.shape[0], 3, "conv2DSS: #shares")
        # conv2DOneFilter :573-580: a filter whose polynomials are all zero is an error
        # (the verdict is read after the layer's kernels are enqueued; on error the outputs are dropped)
        nz = getattr(filters, "_mm_nonzero", None)
        if nz is None:  # polynomials that did not come from encodeFilters: look at them
            nz = L.DeferredFlag((filters.reshape(meta.n_filters, -1) != 0).any(dim=1).all())
        out_cts = self.ctx._empty(p.n_out, 2, 1, self.ctx.N)
        out_share = self.ctx._empty(*p.out_shape)
        self._check_rand(p, rand, ("flood", "u", "e0", "e1", "mask") if exact else ("u", "e1", "mask"))
        if meta.is_shared_input:
            self._need(tuple(img_share1.shape) == (p.n_in, self.ctx.N), 3, "conv2DSS: share plaintexts shape")
        if exact:
            flood, u, e0, e1, mask = rand
            L.check(self.ctx.lib.mmh_conv_server_exact(p.handle, L.dptr(img_share0),
                                                       L.dptr(img_share1 if meta.is_shared_input else None),
                                                       L.dptr(filters), L.dptr(self.pk_last), L.dptr(flood),
                                                       L.dptr(u), L.dptr(e0), L.dptr(e1), L.dptr(mask),
                                                       L.dptr(out_cts), L.dptr(out_share), L._stream_ptr()))
        else:
            u, e1, mask = rand
            L.check(self.ctx.lib.mmh_conv_server(p.handle, L.dptr(img_share0),
                                                 L.dptr(img_share1 if meta.is_shared_input else None),
                                                 L.dptr(filters), L.dptr(self.pk_last), L.dptr(u), L.dptr(e1),
                                                 L.dptr(mask), L.dptr(out_cts), L.dptr(out_share), L._stream_ptr()))
        self._need(bool(nz), 8, "conv2DOneFilter: filter with all zero is not supported")
        return out_cts, out_share

    # encodeFilters + conv2DSS as CheetahLinear::conv2d chains them (cheetah-api.cpp:417-445), in one
    # device call from the raw filters [M, C, fh, fw]; bit-identical to the two-call form
    def conv2DSSFromWeights(self, img_share0, img_share1, filters, meta, rand):
        self._need(self.pk_ntt is not None, 1, "conv2DSS: no public key")
        self._need(filters.shape[0] > 0 and filters.shape[0] == meta.n_filters, 7, "encodeFilters: #filters")
        self._need(tuple(filters.shape[1:]) == tuple(meta.fshape), 3, "encodeFilters: filter shape")
        p = self.plan(meta)
        self._need(tuple(img_share0.shape) == (p.n_in, 2, self.ctx.L, self.ctx.N), 3, "conv2DSS: #ciphertexts")
        if meta.is_shared_input:
            self._need(img_share1 is not None and img_share1.shape[0] == img_share0.shape[0], 3, "conv2DSS: #shares")
        filters = filters.contiguous()
        bad = torch_empty_flag(filters)
        L.check(self.ctx.lib.mmh_conv_check_filters(p.handle, L.dptr(filters), L.dptr(bad), L._stream_ptr()))
        nz = L.DeferredFlag(bad, negate=True)   # true when no filter is all zero
        self._check_rand(p, rand, ("u", "e1", "mask"))
        if meta.is_shared_input:
            self._need(tuple(img_share1.shape) == (p.n_in, self.ctx.N), 3, "conv2DSS: share plaintexts shape")
        u, e1, mask = rand
        out_cts = self.ctx._empty(p.n_out, 2, 1, self.ctx.N)
        out_share = self.ctx._empty(*p.out_shape)
        L.check(self.ctx.lib.mmh_conv_server_weights(p.handle, L.dptr(img_share0),
                                                     L.dptr(img_share1 if meta.is_shared_input else None),
                                                     L.dptr(filters.contiguous()), L.dptr(self.pk_last), L.dptr(u),
                                                     L.dptr(e1), L.dptr(mask), L.dptr(out_cts), L.dptr(out_share),
                                                     L._stream_ptr()))
        self._need(bool(nz), 8, "conv2DOneFilter: filter with all zero is not supported")
        return out_cts, out_share

    # encodeImage + encodeFilters + conv2DSS as CheetahLinear::conv2d chains them (cheetah-api.cpp:401-445), in one
    # device call from the raw tensors: the server's share [C, H, W] (None when the input is not shared) and the
    # filters [M, C, fh, fw]; bit-identical to the three-call form
    def conv2DSSFromTensors(self, img_share0, share_tensor, filters, meta, rand, inline_verdict=False, out=None,
                            defer_verdict=False):
        """out: optional (out_cts [n_out,2,1,N], out_share out_shape) buffers to write into instead of fresh ones
        (pre-sized assembly buffers of the sharded form, openmm_amd/sharding.py).
        The zero-filter rule (conv2DOneFilter :573-580) is evaluated inside the call; by default its verdict is read
        early, from page-locked memory behind the call's second launch (mmh_conv_server_tensors_ev), so the host
        raises the reference's error without waiting for the products.  inline_verdict: the older form, the verdict
        in device memory and read when the whole call has run.  defer_verdict: the call returns without waiting at
        all and the verdict is read by raise_pending() behind the caller's own synchronisation -- what the C++ host
        does (it synchronises once per layer anyway, before the send: openmm_amd/host/cheetah_linear.cc) and what a
        caller that enqueues many layers ahead wants; at most 256 calls may be pending.
        rand: (u, e1, mask) tensors, or an openmm_amd.lib.Sampler: the call then draws the three itself, from the next
        three streams of that sampler -- the same values sampler.reshare(n_out) would have returned."""
        self._need(self.pk_ntt is not None, 1, "conv2DSS: no public key")
        self._need(filters.shape[0] > 0 and filters.shape[0] == meta.n_filters, 7, "encodeFilters: #filters")
        self._need(tuple(filters.shape[1:]) == tuple(meta.fshape), 3, "encodeFilters: filter shape")
        p = self.plan(meta)
        self._need(tuple(img_share0.shape) == (p.n_in, 2, self.ctx.L, self.ctx.N), 3, "conv2DSS: #ciphertexts")
        if meta.is_shared_input:
            self._need(share_tensor is not None and tuple(share_tensor.shape) == tuple(meta.ishape), 3,
                       "encodeImage: image shape")
            share_tensor = share_tensor.contiguous()
        filters = filters.contiguous()
        drawn = isinstance(rand, L.Sampler)   # the call draws u, e1 and the mask itself (mmh_conv_server_tensors_sampled)
        if not drawn:
            self._check_rand(p, rand, ("u", "e1", "mask"))
            u, e1, mask = rand
        if out is None:
            out_cts = self.ctx._empty(p.n_out, 2, 1, self.ctx.N)
            out_share = self.ctx._empty(*p.out_shape)
        else:
            out_cts, out_share = out
            self._need(tuple(out_cts.shape) == (p.n_out, 2, 1, self.ctx.N) and tuple(out_share.shape) == p.out_shape,
                       3, "conv2DSS: output buffers")
        share_ptr = L.dptr(share_tensor if meta.is_shared_input else None)
        if drawn:
            if self._verdicts is None:
                self._verdicts = L.VerdictRing(256)
            self._need(len(self._pending) < 255, 5, "conv2DSS: too many deferred verdicts, call raise_pending()")
            slot, word, event = self._verdicts.take()
            L.check(self.ctx.lib.mmh_conv_server_tensors_sampled(p.handle, L.dptr(img_share0), share_ptr, L.dptr(filters),
                                                                 L.dptr(self.pk_last), rand.key, rand.reshare_streams(), 0,
                                                                 L.dptr(out_cts), L.dptr(out_share), word, event,
                                                                 L._stream_ptr()))
            if defer_verdict:
                self._pending.append(slot)
                return out_cts, out_share
            nz = self._verdicts.read(slot) == 0
        elif inline_verdict:
            bad = torch_empty_flag(filters)   # zero-filter verdict, known when the whole call has run
            L.check(self.ctx.lib.mmh_conv_server_tensors(p.handle, L.dptr(img_share0), share_ptr, L.dptr(filters),
                                                         L.dptr(self.pk_last), L.dptr(u), L.dptr(e1), L.dptr(mask),
                                                         L.dptr(out_cts), L.dptr(out_share), L.dptr(bad),
                                                         L._stream_ptr()))
            nz = bool(L.DeferredFlag(bad, negate=True))
        else:
            # the verdict lands in page-locked memory behind the call's second launch; wait for that point alone
            if self._verdicts is None:
                self._verdicts = L.VerdictRing(256)
            self._need(len(self._pending) < 255, 5, "conv2DSS: too many deferred verdicts, call raise_pending()")
            slot, word, event = self._verdicts.take()
            L.check(self.ctx.lib.mmh_conv_server_tensors_ev(p.handle, L.dptr(img_share0), share_ptr, L.dptr(filters),
                                                            L.dptr(self.pk_last), L.dptr(u), L.dptr(e1), L.dptr(mask),
                                                            L.dptr(out_cts), L.dptr(out_share), word, event,
                                                            L._stream_ptr()))
            if defer_verdict:
                self._pending.append(slot)
                return out_cts, out_share
            nz = self._verdicts.read(slot) == 0   # true when no filter is all zero
        self._need(nz, 8, "conv2DOneFilter: filter with all zero is not supported")
        return out_cts, out_share

    def raise_pending(self):
        """Behind a synchronisation of the stream: the zero-filter verdicts of the calls made with defer_verdict since
        the last time; raises the reference's error if any of them saw an all-zero filter."""
        slots, self._pending = self._pending, []
        bad = [i for i in slots if int(self._verdicts.words[i]) != 0]
        self._need(not bad, 8, "conv2DOneFilter: filter with all zero is not supported")

    # static weights: encode once per model, then conv2DSSPrepared per inference (same bits as
    # conv2DSSFromWeights); the zero-filter rule of conv2DOneFilter :573-580 is settled here
    def prepareFilters(self, filters, meta):
        self._need(filters.shape[0] > 0 and filters.shape[0] == meta.n_filters, 7, "encodeFilters: #filters")
        self._need(tuple(filters.shape[1:]) == tuple(meta.fshape), 3, "encodeFilters: filter shape")
        nz = bool((_mod_t(filters, self.ctx.t) != 0).reshape(meta.n_filters, -1).any(dim=1).all())
        self._need(nz, 8, "conv2DOneFilter: filter with all zero is not supported")
        return PreparedFilters(self.plan(meta), filters, nz)

    def conv2DSSPrepared(self, img_share0, img_share1, prepared, meta, rand, share_tensor=None):
        """share_tensor: the server's share as the raw tensor instead of its encoding img_share1 (encodeImage fused
        into the call)"""
        self._need(self.pk_ntt is not None, 1, "conv2DSS: no public key")
        p = self.plan(meta)
        self._need(prepared.plan is p, 7, "conv2DSS: filters prepared for another layer")
        self._need(tuple(img_share0.shape) == (p.n_in, 2, self.ctx.L, self.ctx.N), 3, "conv2DSS: #ciphertexts")
        raw = share_tensor is not None
        if meta.is_shared_input and raw:
            self._need(img_share1 is None and tuple(share_tensor.shape) == tuple(meta.ishape), 3, "encodeImage: image shape")
            share_tensor = share_tensor.contiguous()
        elif meta.is_shared_input:
            self._need(img_share1 is not None and img_share1.shape[0] == img_share0.shape[0], 3, "conv2DSS: #shares")
            self._need(tuple(img_share1.shape) == (p.n_in, self.ctx.N), 3, "conv2DSS: share plaintexts shape")
        self._check_rand(p, rand, ("u", "e1", "mask"))
        u, e1, mask = rand
        out_cts = self.ctx._empty(p.n_out, 2, 1, self.ctx.N)
        out_share = self.ctx._empty(*p.out_shape)
        fn = self.ctx.lib.mmh_conv_server_prepared_tensors if raw else self.ctx.lib.mmh_conv_server_prepared
        share = (share_tensor if raw else img_share1) if meta.is_shared_input else None
        L.check(fn(p.handle, L.dptr(img_share0), L.dptr(share), prepared.handle, L.dptr(self.pk_last), L.dptr(u),
                   L.dptr(e1), L.dptr(mask), L.dptr(out_cts), L.dptr(out_share), L._stream_ptr()))
        return out_cts, out_share

    # the re-sharing tail split at the point where the input enters it (include/mm_hip.h): the encryptions of zero
    # under addRandomMask (hom_conv2d_ss.cc:769, :275-340) made ahead of the inputs, the layer call then online only
    def prepareZeros(self, meta, u):
        """u [n_out, N] ternary -> [n_out, 2, N]: u * pk_j in coefficient form at the last level"""
        self._need(self.pk_ntt is not None, 1, "conv2DSS: no public key")
        p = self.plan(meta)
        self._need(tuple(u.shape) == (p.n_out, self.ctx.N) and u.element_size() == 8, 3, "prepareZeros: u shape")
        zero = self.ctx._empty(p.n_out, 2, self.ctx.N)
        L.check(self.ctx.lib.mmh_reshare_zero_prepare(self.ctx.handle, L.dptr(self.pk_last), L.dptr(u.contiguous()),
                                                      p.n_out, L.dptr(zero), L._stream_ptr()))
        return zero

    def conv2DSSOnline(self, img_share0, share_tensor, prepared, zeros, meta, rand):
        """conv2DSSPrepared with the encryptions of zero from prepareZeros and the share as the raw tensor
        (encodeImage fused into the call, as conv2DSSFromTensors does); rand = (e1, mask)"""
        p = self.plan(meta)
        self._need(prepared.plan is p, 7, "conv2DSS: filters prepared for another layer")
        self._need(tuple(img_share0.shape) == (p.n_in, 2, self.ctx.L, self.ctx.N), 3, "conv2DSS: #ciphertexts")
        self._need(tuple(zeros.shape) == (p.n_out, 2, self.ctx.N), 3, "conv2DSS: prepared zeros shape")
        if meta.is_shared_input:
            self._need(share_tensor is not None and tuple(share_tensor.shape) == tuple(meta.ishape), 3,
                       "encodeImage: image shape")
            share_tensor = share_tensor.contiguous()
        self._check_rand(p, rand, ("e1", "mask"))
        e1, mask = rand
        out_cts = self.ctx._empty(p.n_out, 2, 1, self.ctx.N)
        out_share = self.ctx._empty(*p.out_shape)
        L.check(self.ctx.lib.mmh_conv_server_online(p.handle, L.dptr(img_share0), L.dptr(None),
                                                    L.dptr(share_tensor if meta.is_shared_input else None),
                                                    prepared.handle, L.dptr(zeros), L.dptr(e1), L.dptr(mask),
                                                    L.dptr(out_cts), L.dptr(out_share), L._stream_ptr()))
        return out_cts, out_share

    # decryptToTensor (hom_conv2d_ss.cc:853-941)
    def decryptToTensor(self, enc_tensor, meta):
        self._need(self.sk_ntt is not None, 1, "decrypt without sk")
        p = self.plan(meta)
        self._need(enc_tensor.shape[0] == p.n_out, 8, "decryptToTensor: #ciphertexts")
        out = self.ctx._empty(*p.out_shape)
        L.check(self.ctx.lib.mmh_conv_decrypt(p.handle, L.dptr(self.sk_last), L.dptr(enc_tensor), L.dptr(out),
                                              L._stream_ptr()))
        return out

    # compact wire form of the result ciphertexts (what seal::Ciphertext::save's compression does for the
    # reference, cheetah-api.cpp:11-29): [n_out][words_per_ct] words, unpack(pack(cts)) == cts
    def packedWords(self, meta):
        n = C.c_size_t()
        L.check(self.ctx.lib.mmh_conv_result_packed_words(self.plan(meta).handle, C.byref(n)))
        return n.value

    def packResult(self, enc_tensor, meta):
        p = self.plan(meta)
        self._need(tuple(enc_tensor.shape) == (p.n_out, 2, 1, self.ctx.N), 3, "packResult: ciphertext shape")
        out = self.ctx._empty(p.n_out, self.packedWords(meta))
        L.check(self.ctx.lib.mmh_conv_result_pack(p.handle, L.dptr(enc_tensor.contiguous()), L.dptr(out),
                                                  L._stream_ptr()))
        return out

    def unpackResult(self, packed, meta):
        p = self.plan(meta)
        self._need(tuple(packed.shape) == (p.n_out, self.packedWords(meta)), 3, "unpackResult: packed shape")
        out = self.ctx._empty(p.n_out, 2, 1, self.ctx.N)
        L.check(self.ctx.lib.mmh_conv_result_unpack(p.handle, L.dptr(packed.contiguous()), L.dptr(out),
                                                    L._stream_ptr()))
        return out

    # idealFunctionality (hom_conv2d_ss.cc:975-1012; Tensor::Conv2D tensor.h:274-362), mod 2^k only
    def idealFunctionality(self, in_tensor, filters, meta):
        import torch
        t = self.ctx.t
        C_, H, W = meta.ishape
        fh, fw = meta.fshape[1:]
        ph = (fh - 1) if meta.padding == SAME else 0
        pw = (fw - 1) if meta.padding == SAME else 0
        top, left = (ph + 1) // 2, (pw + 1) // 2
        x = torch.zeros((C_, H + ph, W + pw), dtype=torch.int64, device=in_tensor.device)
        x[:, top:top + H, left:left + W] = in_tensor
        oh, ow = (H + ph - fh + meta.stride) // meta.stride, (W + pw - fw + meta.stride) // meta.stride
        out = torch.zeros((meta.n_filters, oh, ow), dtype=torch.int64, device=in_tensor.device)
        for r in range(fh):
            for c in range(fw):
                patch = x[:, r:r + (oh - 1) * meta.stride + 1:meta.stride, c:c + (ow - 1) * meta.stride + 1:meta.stride]
                out += (filters[:, :, r, c, None, None] * patch[None]).sum(1)  # int64 wraps mod 2^64
        return out & (t - 1) if t & (t - 1) == 0 else out
