"""Rotary positions on secret shares.

The turn's coefficients are public, so each party turns its own share: with fixed-point c + i s = 2^f exp(i angle) the pair
(a, b) becomes (a c - b s, b c + a s) modulo 2^l, and a truncation by f (``Truncation.truncate_rotary``) takes the scale off
again.  Both parties must use the same coefficients to the last bit; they are functions of the phase steps below, which are
integers computed with decimal arithmetic and do not depend on a machine's mathematics library.
"""
from decimal import Decimal, localcontext

import torch

from . import lib as L
from .ring_fc_ss import _need
from .truncation import ALICE, BOB

_INT64 = torch.int64
_stream_of, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def rotary_phases(rot_dim, base=10000, linear=1, ntk=1, yarn=None):
    """Phase steps of the rot_dim / 2 pairs: round(2^64 * theta_i / (2 pi)) with theta_i = base^(-2 i / rot_dim), as Python
    integers below 2^64.  For contexts longer than the model was trained for (one of them, or none):

    linear: positions are divided by this factor (theta_i / linear)
    ntk: the base is multiplied by ntk^(rot_dim / (rot_dim - 2)), which leaves the fastest pair and divides the slowest by ntk
    yarn: (factor, trained_length) or (factor, trained_length, slow, fast), where slow = 1 and fast = 32 if not given: pairs that
        make fewer than ``slow`` turns over the trained length are divided by the factor, those with more than ``fast`` are
        left, those between are blended linearly in the number of turns.  (The usual amplitude for it is 1 + ln(factor) / 10.)"""
    _need(rot_dim >= 0 and rot_dim % 2 == 0, 3, "rotary_phases: rot_dim")
    _need(base > 0 and linear > 0 and ntk > 0, 7, "rotary_phases: base or factor")
    _need((linear != 1) + (ntk != 1) + (yarn is not None) <= 1, 7, "rotary_phases: one scaling at a time")
    _need(ntk == 1 or rot_dim > 2, 7, "rotary_phases: ntk needs two pairs")
    _need(yarn is None or len(yarn) in (2, 4), 7, "rotary_phases: yarn")
    out = []
    with localcontext() as ctx:
        ctx.prec = 50
        b = Decimal(base)
        if ntk != 1:
            b *= (Decimal(ntk).ln() * Decimal(rot_dim) / Decimal(rot_dim - 2)).exp()
        for i in range(rot_dim // 2):
            turns = (b.ln() * Decimal(-2 * i) / Decimal(rot_dim)).exp() / (2 * _PI) / Decimal(linear)   # per position
            if yarn is not None:
                factor, length = Decimal(yarn[0]), Decimal(yarn[1])
                slow, fast = (Decimal(yarn[2]), Decimal(yarn[3])) if len(yarn) == 4 else (Decimal(1), Decimal(32))
                _need(factor > 0 and length > 0 and fast > slow, 7, "rotary_phases: yarn")
                keep = min(Decimal(1), max(Decimal(0), (turns * length - slow) / (fast - slow)))
                turns = turns * keep + turns / factor * (1 - keep)
            out.append(int((turns * (1 << 64)).to_integral_value()) % (1 << 64))
    return out


class Rotary:
    """Rotary(phases, head_dim, frac_bits, ring_bw): turns shares x [tokens, heads, head_dim] (any strides over tokens and
    heads, words of a head contiguous) by positions int64 [tokens].  ``phases``: the integers of ``rotary_phases`` or an int64
    CUDA tensor with their bits; 2 * len(phases) <= head_dim words of each head are turned, the others are multiplied by
    2^frac_bits.  Pairs are (i, i + len(phases)), or (2i, 2i + 1) when interleaved."""

    def __init__(self, phases, head_dim, frac_bits, ring_bw, interleaved=False, amplitude=1.0, device="cuda:0"):
        self.lib = L.load_library()
        if not isinstance(phases, torch.Tensor):
            phases = torch.tensor([p - (1 << 64) if p >= 1 << 63 else p for p in phases], dtype=torch.int64, device=device)
        _need(phases.is_cuda and phases.dtype == torch.int64 and phases.dim() == 1 and phases.is_contiguous(), 7,
              "Rotary: expected a contiguous 1-D int64 CUDA tensor of phases")
        _need(head_dim >= 1 and 2 * phases.numel() <= head_dim, 3, "Rotary: more pairs than a head has")
        _need(2 <= ring_bw <= 64 and 0 <= frac_bits <= 24 and 0 < amplitude <= 16, 7, "Rotary: ring_bw, frac_bits or amplitude")
        self.phases, self.head_dim, self.frac_bits, self.ring_bw = phases, head_dim, frac_bits, ring_bw
        self.interleaved, self.amplitude = bool(interleaved), float(amplitude)

        self._dev = phases.get_device()
        self._pairs = (phases.data_ptr(), 2 * phases.numel(), self.interleaved, self.amplitude, self.frac_bits, self.ring_bw)

    def _strides(self, x):
        if x.dtype is not _INT64 or x.dim() != 3 or x.get_device() != self._dev:
            raise L.MMHError(7, "Rotary: expected a 3-D int64 tensor [tokens, heads, head_dim] on the phases' device")
        if x.shape[2] != self.head_dim:
            raise L.MMHError(3, "Rotary: head_dim")
        token, head, word = x.stride()
        if word != 1 and self.head_dim != 1 and x.numel():
            raise L.MMHError(7, "Rotary: the words of a head must be contiguous")
        return token, head

    def _args(self, x, positions):
        token, head = self._strides(x)
        if positions.dtype is not _INT64 or positions.dim() != 1 or positions.get_device() != self._dev or \
                not positions.is_contiguous():
            raise L.MMHError(7, "Rotary: expected contiguous int64 positions on the phases' device")
        tokens, heads, dim = x.shape
        if positions.shape[0] != tokens:
            raise L.MMHError(3, "Rotary: #positions")
        return (x.data_ptr(), token, head, tokens, heads, dim, positions.data_ptr()) + self._pairs

    def _check_apart(self, out, token, head, args):
        px, xt, xh, tokens, heads, dim, pos, phase, rot = args[:9]
        po = out.data_ptr()
        if not (tokens and heads):
            return
        end = po + 8 * ((tokens - 1) * token + (heads - 1) * head + dim)
        mine = (po, dim, ((tokens, token), (heads, head)))
        operands = [(pos, 0, 0, 1, 1, tokens), (phase, 0, 0, 1, 1, rot // 2)]
        if not (px == po and (xt == token or tokens == 1) and (xh == head or heads == 1)):
            operands.append((px, xt, xh, tokens, heads, dim))
        for p, t, h, n, m, width in operands:
            if p < end and po < p + 8 * ((n - 1) * t + (m - 1) * h + width):
                _need(not L.rows_overlap(mine, (p, width, ((n, t), (m, h)))), 7, "Rotary: out overlaps an operand")

    def _call(self, fn, args):
        args += (_stream_of(self._dev),)
        if _current_device() == self._dev:
            rc = fn(*args)
        else:
            with torch.cuda.device(self._dev):
                rc = fn(*args)
        if rc:
            L.check(rc)

    def rotate(self, x, positions, out=None):
        """the turned share, scaled by 2^frac_bits; ``out`` may be x (same strides), or another tensor of the shape that shares
        no word with x, positions or phases"""
        args = self._args(x, positions)
        if out is None:
            out = x.new_empty(x.shape)
            token, head = args[4] * args[5], args[5]
        else:
            token, head = self._strides(out)
            _need(out.shape == x.shape, 3, "Rotary: out")
            self._check_apart(out, token, head, args)
        self._call(self.lib.mmh_rotary, args + (out.data_ptr(), token, head))
        return out

    def truncate_pre(self, party, x, positions, signed_arithmetic=True, apply_msb0_heuristic=True):
        """the turned share as the truncation's wrap protocol takes it, and the operand of its comparison (None with the
        heuristic, which does not compare)"""
        _need(party in (ALICE, BOB), 7, "Rotary: party")
        args = self._args(x, positions)
        adj = x.new_empty(x.shape)
        cmp = None if apply_msb0_heuristic else torch.empty_like(adj)
        self._call(self.lib.mmh_rotary_trunc_pre, (party,) + args + (bool(signed_arithmetic), bool(apply_msb0_heuristic),
                                                                     adj.data_ptr(), 0 if cmp is None else cmp.data_ptr()))
        return adj, cmp
