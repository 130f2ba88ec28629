"""Rotary positions on encrypted queries and keys (no counterpart in the reference: its application rotates before it encrypts).

Position p turns pair j of every head by theta_j = p[axis[j]] * inv_freq[j]; with several axes (time, height, width of a video's
patches) each pair follows one of them. Heads lie in the slots as compute_qkt reads them (src/attention.cu:10-28): slot
t * heads * d_head + h * d_head + i of a ciphertext holds element i of head h at its t-th position.

  packing "pairs"        a slot holds x + i y of a pair (what matrices folded into complex ones deliver): one product with
                         exp(i theta), no key switch. q . k is then the real part of the sum over q' conj(k'): conjugate k' once
                         (`rotate(ct, 0)`) as it goes into the cache.
  packing "halves"       real slots, pair j = elements j and j + pairs; x C + rot(x, s) A + rot(x, -s) B with s = pairs
  packing "interleaved"  the same with pair j = elements 2 j and 2 j + 1, s = 1: two rotations from one decomposition

Elements of a head beyond its pairs pass unchanged. Positions that are dropped (`keep`), and slots of no position, come out as zeros:
a decoding step's one position goes into its place of a page that way, without a mask of its own.
"""
import math
from array import array

import torch

from . import _operands, hoist_rotations, plaintext
from ._native import LIB, check, current_stream as _stream, on_device

_PACKINGS = {"pairs": 0, "halves": 1, "interleaved": 2}
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}
CHUNK = 16  # ciphertexts whose encodings, products and rescales go together; rotations take them one after another


class rotary:
    def __init__(self, context, inv_freq, heads, d_head, axes=None, packing="pairs", scaling=1.0):
        """inv_freq: the angle per position of each pair (a sequence or a tensor); axes: the axis of each pair, 0 if not given;
        scaling: a factor on sines and cosines"""
        if packing not in _PACKINGS:
            raise ValueError("rotary: packing is 'pairs', 'halves' or 'interleaved'")
        f = torch.as_tensor(inv_freq, dtype=torch.float64).reshape(-1).to(device=context.device).clone()
        heads, d_head, pairs = int(heads), int(d_head), f.numel()
        if heads < 1 or d_head < 1 or heads * d_head > context.N // 2:
            raise ValueError("rotary: heads * d_head must be in [1, slots]")
        if pairs < 1 or pairs > (d_head if packing == "pairs" else d_head // 2):
            raise ValueError("rotary: more pairs than a head holds")
        angles = f.tolist()
        if not (math.isfinite(scaling) and all(math.isfinite(v * 2.0 ** 64) for v in angles)):  # the angle of any integer position
            raise ValueError("rotary: the angles per position and the scaling must be finite (below 2^960)")
        a = [0] * pairs if axes is None else [int(v) for v in axes]
        if len(a) != pairs or min(a) < 0:
            raise ValueError("rotary: an axis for every pair is wanted")
        self.ctx, self.heads, self.d_head, self.pairs, self.packing, self.scaling = context, heads, d_head, pairs, packing, float(scaling)
        self.n_axes = max(a) + 1
        self.positions_per_ct = context.N // 2 // (heads * d_head)
        self.inv_freq, self.axes = f, torch.tensor(a, dtype=torch.int32, device=context.device)
        steepest = {}  # the largest angle per position on each axis that a pair follows
        for axis, angle in zip(a, angles):
            steepest[axis] = max(steepest.get(axis, 0.0), abs(angle))
        self._followed, self._steepest = torch.tensor(list(steepest), device=f.device), torch.tensor(list(steepest.values()), dtype=torch.float64, device=f.device)
        self.step = pairs if packing == "halves" else 1
        self._vecs = 1 if packing == "pairs" else 3
        torch.cuda.synchronize(context.device)  # the tables are there for whichever stream comes first

    def factors(self, positions, keep=None, conjugate=False):
        """The factors of `positions` ([tokens] or [tokens][axes], int32, int64, float32 or float64, any strides) as complex128
        [vectors][ciphertexts][slots], one vector ("pairs") or three (C, A, B), positions_per_ct tokens to a ciphertext. keep: bool
        [tokens], False for a token whose slots become zeros. conjugate: the inverse rotation."""
        ctx, p, dims = self.ctx, positions, positions.dim()
        kind = _POSITIONS.get(p.dtype)
        if not 1 <= dims <= 2 or kind is None:
            raise ValueError("rotary: positions are [tokens] or [tokens][axes] of int32, int64, float32 or float64")
        tokens = p.shape[0]
        if (p.shape[1] if dims == 2 else 1) < self.n_axes:
            raise ValueError("rotary: positions have fewer axes than the pairs name")
        if keep is not None and (keep.dtype != torch.bool or keep.dim() != 1 or keep.shape[0] != tokens):
            raise ValueError("rotary: keep is one truth value a token")
        if p.get_device() != ctx.device or (keep is not None and keep.get_device() != ctx.device):
            raise ValueError("rotary: positions and keep must lie on the context's device")
        if p.is_neg():  # the imaginary part of a conjugate: its words are not its values
            p = p.resolve_neg()
        out = torch.empty(self._vecs, -(-tokens // self.positions_per_ct), ctx.N // 2, dtype=torch.complex128, device=ctx.device)
        with on_device(ctx):
            check(LIB.b2_rotary_factors(ctx._h, _PACKINGS[self.packing], tokens, self.heads, self.d_head, self.pairs, p.data_ptr(), kind, p.stride(0),
                                        p.stride(1) if dims == 2 else 0, self.inv_freq.data_ptr(), self.axes.data_ptr(), 0 if keep is None else keep.data_ptr(),
                                        0 if keep is None else keep.stride(0), self.scaling, 1 if conjugate else 0, out.data_ptr(), _stream()))
        return out

    def encode(self, encoder, factors, chain_index):
        """[vector][ciphertext] plaintexts of `factors` at a level, at the scale of the prime that the rescale after the product
        removes. Queries and keys of all layers at that level and of these positions share them. Values too large for a plaintext,
        and what is no finite number, are refused; for that the host waits for the factors. While a graph is captured it cannot, and
        takes them as they are."""
        return self._encode(encoder, factors, chain_index, False)

    def _encode(self, encoder, factors, chain_index, made_here):
        """made_here: the values are this object's, of finite positions"""
        ctx = self.ctx
        if factors.dim() != 3 or factors.dtype != torch.complex128 or factors.shape[2] != ctx.N // 2:
            raise ValueError("rotary: factors are complex128 [vectors][ciphertexts][slots]")
        if encoder.ctx is not ctx:
            raise ValueError("rotary: the encoder belongs to another context")
        if chain_index < 1:
            raise ValueError("chain index out of range")
        l = ctx.limbs_at(chain_index)
        if l < 2:
            raise ValueError("end of modulus switching chain reached")
        scale = float(ctx.primes[l - 1])
        if scale * max(1.0, abs(self.scaling)) * 1.4143 >= 2.0 ** 61:  # no coefficient exceeds it, and none may pass 62 bits
            raise ValueError("scale out of bounds")
        vecs, n = factors.shape[0], factors.shape[1]
        if vecs == 0 or n == 0:
            return [[] for _ in range(vecs)]
        vals = factors.to(device=ctx.device).clone(memory_format=torch.contiguous_format)  # overwritten by the transform
        coeffs, data = torch.empty(vecs * n, ctx.N, dtype=torch.int64, device=ctx.device), ctx.empty(vecs, n, l)
        with on_device(ctx):
            largest = max(1.0, abs(self.scaling))
            if not made_here and not torch.cuda.is_current_stream_capturing():
                low, high = torch.view_as_real(vals).aminmax()
                largest = float(torch.maximum(-low, high))  # NaN if there is one
            bound = 1.4143 * largest * scale
            if not (bound < 2.0 ** 61 and math.log2(max(bound, 1.0)) + 2 < ctx.chain_bits[l]):
                raise ValueError("encoded values are too large")
            check(LIB.b2_encode_coeffs_batch(ctx._h, vecs * n, vals.data_ptr(), encoder._d_rot.data_ptr(), encoder._d_ksi.data_ptr(), scale / encoder.slots,
                                             coeffs.data_ptr(), _stream()))
            check(LIB.b2_expand_single_chain_batch(ctx._h, l, vecs * n, coeffs.data_ptr(), data.data_ptr(), _stream()))
        return [[self._plain(data[v, i], chain_index, l, scale) for i in range(n)] for v in range(vecs)]

    def _plain(self, data, chain_index, l, scale):
        pt = plaintext()
        pt._chain_index, pt._N, pt._limbs, pt._scale, pt.data = chain_index, self.ctx.N, l, scale, data
        return pt

    def apply(self, xs, plaintexts, galois_key=None):
        """the ciphertexts xs (of one level and scale) rotated by the encoded factors, one level further down (rounded to nearest), at
        their scale: the plaintexts are at the prime's that the rescale removes, as `encode` makes them, and at no other. "halves" and
        "interleaved" want Galois keys for the steps +-`step`."""
        ctx, vecs = self.ctx, self._vecs
        if len(plaintexts) != vecs or any(len(v) != len(xs) for v in plaintexts):
            raise ValueError("rotary: as many encoded factors as ciphertexts are wanted")
        if not len(xs):
            return []
        if vecs == 3 and galois_key is None:
            raise ValueError("Galois key not present")
        first, _, _ = _operands(ctx, [xs])
        l = first._limbs
        if any(pt._chain_index != first._chain_index or pt.data.shape != (l, ctx.N) or pt.data.dtype != torch.int64 or pt.data.get_device() != ctx.device
               for v in plaintexts for pt in v):
            raise ValueError("encrypted and plain parameter mismatch")
        if l < 2:
            raise ValueError("end of modulus switching chain reached")
        prime = float(ctx.primes[l - 1])
        if not all(abs(pt._scale - prime) <= 1e-9 * prime for v in plaintexts for pt in v):
            raise ValueError("scale mismatch")
        out = []
        with on_device(ctx):
            for i in range(0, len(xs), CHUNK):
                out += self._apply(xs[i:i + CHUNK], [v[i:i + CHUNK] for v in plaintexts], galois_key, l)
        return out

    def _apply(self, xs, plaintexts, galois_key, l):
        ctx, n, first = self.ctx, len(xs), xs[0]
        # rotations read dense polynomials: of a view (the first limbs of a higher level) a dense copy is rotated and multiplied
        xs = [x if x.data.is_contiguous() else x._like(x.data.contiguous().view(2, l, ctx.N)) for x in xs]
        terms = [[x] for x in xs] if self._vecs == 1 else [[x] + hoist_rotations(ctx, x, galois_key, [self.step, -self.step]) for x in xs]
        _, cts, held = _operands(ctx, terms)
        factors = [pt.data.contiguous() for i in range(n) for pt in (v[i] for v in plaintexts)]
        pts = array("Q", [t.data_ptr() for t in factors])
        y, out, ws = ctx.empty(n, 2, l), ctx.empty(n, 2, l - 1), ctx.empty(2 * n)
        check(LIB.b2_multiply_plain_sum(ctx._h, l, n, self._vecs, cts.buffer_info()[0], pts.buffer_info()[0], y.data_ptr(), _stream()))
        check(LIB.b2_rescale_rounded_batch(ctx._h, l, n, y.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel() * 8, _stream()))
        return [first._like(z, chain_index=first._chain_index + 1, scale=x._scale) for x, z in zip(xs, out.unbind(0))]

    def forward(self, encoder, xs, positions, keep=None, conjugate=False, galois_key=None):
        """factors, encode and apply for ciphertexts of one level, CHUNK of them at a time. A kept position that is not finite would
        spoil its whole ciphertext and is refused; for that the host waits for positions in floating point, except while a graph is
        captured."""
        f = self.factors(positions, keep, conjugate)
        if f.shape[1] != len(xs):
            raise ValueError("rotary: positions for ceil(tokens / positions_per_ct) ciphertexts were given")
        self._check_finite(positions, keep)
        out = []
        for i in range(0, len(xs), CHUNK):
            part = xs[i:i + CHUNK]
            if any(x._chain_index != part[0]._chain_index for x in part):
                raise ValueError("encrypted and plain parameter mismatch")
            out += self.apply(part, self._encode(encoder, f[:, i:i + CHUNK], part[0]._chain_index, True), galois_key)
        return out

    def _check_finite(self, positions, keep):
        if not positions.dtype.is_floating_point:  # every integer's angle is
            return
        with on_device(self.ctx):
            if torch.cuda.is_current_stream_capturing():
                return
            p = (positions if positions.dim() == 2 else positions[:, None])[:, self._followed].double()
            bad = ~torch.isfinite(p * self._steepest).all(1)
            if bool((bad if keep is None else bad & keep).any()):
                raise ValueError("rotary: a kept position is not finite")
