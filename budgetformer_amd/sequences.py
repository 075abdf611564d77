"""Operators over packed sequences: softmax attention, rotary positions, linear attention with decay.

Sequences lie one behind the other along the first dimension of [rows, heads, head_dim] tensors: the node
sequences of a batch of graphs, random walks (a walk is the sequence of its nodes), prompts of different
lengths. ``PackedSequences`` holds what a batch's layers share: where each sequence starts and what each
row sees, built on the GPU once per batch as an ``AttentionIndex`` is once per edge set.

  packed_attention       dense softmax attention inside each sequence (grouped heads, causal or not)
  rotary_embedding       rotary positions of q and k
  linear_attention       linear attention with a decay for each head, chunked; linear_attention_step: its
                         recurrent form for single tokens

``CoreAttention`` takes the first (and, with ``rotary``, the second) for ``attn_type="flash"``, the dense
attention of models/graphormer_dist_node_level.py:603-608. All run as HIP kernels on the current stream;
there is no CPU fallback. Activations are float32, bfloat16 or float16, sums and statistics float32. Gradients
are backward-mode and once differentiable; dual tensors (forward mode) are refused.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _native as N

_MOST_ROWS = 2 ** 31 - 2 ** 17


def _op(name: str):
    """The overload of a ``bf`` operator, resolved once (an operator's own lookup costs a call some 2 us)."""
    got = _OPS.get(name)
    if got is None:
        got = _OPS[name] = getattr(N.load_ops(), name).default
    return got


_OPS: dict = {}


def _raw_stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _as(q: torch.Tensor, t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == q.dtype else t.to(q.dtype)


def _trains(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class PackedSequences:
    """Where the sequences of a packed batch start, and what each row sees.

    Query rows of sequence s are ``[q_offsets[s], q_offsets[s + 1])`` and see keys of
    ``[k_offsets[s], k_offsets[s + 1])``: all of them, or with ``causal`` those up to their own place, the last
    query at the last key (one query a sequence then sees all its keys). Rows behind the last sequence see
    nothing: their outputs and gradients are 0.

    A captured graph reads these tensors at each replay: keep the object as long as the graph.
    """

    # Plain tensors also where a batch is built in inference mode: training later saves them.
    @torch.inference_mode(False)
    def __init__(self, q_offsets: torch.Tensor, k_offsets: torch.Tensor, n_q: int, n_k: int, causal: bool, longest: int = 0):
        if q_offsets.is_inference() or k_offsets.is_inference():
            same = q_offsets is k_offsets
            q_offsets = q_offsets.clone()
            k_offsets = q_offsets if same else k_offsets.clone()
        self.longest = int(longest)          # no sequence has more rows or keys; 0: unknown
        self.q_offsets, self.k_offsets = q_offsets, k_offsets
        self.n_q, self.n_k, self.n_seq, self.causal = int(n_q), int(n_k), q_offsets.numel() - 1, bool(causal)
        self.self_attention = q_offsets is k_offsets and self.n_q == self.n_k
        self.row_span, self.key_span, self._positions = _op("packed_spans")(q_offsets, k_offsets, self.n_q, self.n_k,
                                                                            self.causal)
        # the stream that fills them; others wait for it once (see used)
        self._streams = {_raw_stream(self.device)}
        self._ready = None
        if not torch.cuda.is_current_stream_capturing():
            self._ready = torch.cuda.Event()
            self._ready.record(torch.cuda.current_stream(self.device))

    def used(self) -> None:
        """Before a call on the current stream: if another stream filled the spans, this one waits for them, and
        their memory is not handed out while it may read them."""
        raw = _raw_stream(self.device)
        if raw in self._streams or self._ready is None or torch.cuda.is_current_stream_capturing():
            return
        stream = torch.cuda.current_stream(self.device)
        stream.wait_event(self._ready)
        for t in (self.q_offsets, self.k_offsets, self.row_span, self.key_span, self._positions):
            t.record_stream(stream)
        self._streams.add(raw)

    @staticmethod
    def _sizes(n_q: int, n_k: int) -> None:
        if not (0 <= n_q < _MOST_ROWS and 0 <= n_k < _MOST_ROWS):
            raise ValueError(f"{n_q} query rows and {n_k} keys (below 2^31 - 2^17 each)")

    @classmethod
    def from_lengths(cls, q_lengths: Sequence[int], k_lengths: Optional[Sequence[int]] = None, *, causal: bool = False,
                     device="cuda") -> "PackedSequences":
        """From the sequences' lengths on the host (a list, or a CPU tensor); ``k_lengths``: those of the keys
        where they differ. Nothing is read back from the device. Not under graph capture, which would copy from the host's
        lengths again at each replay (``from_offsets`` without the check)."""
        device = cls._device(device)
        lens = [torch.as_tensor(x, dtype=torch.int64, device="cpu") for x in
                ((q_lengths,) if k_lengths is None else (q_lengths, k_lengths))]
        for x in lens:
            if x.dim() != 1 or x.numel() != lens[0].numel():
                raise ValueError("q_lengths and k_lengths must be one length for each sequence")
            if x.numel() and int(x.min()) < 0:
                raise ValueError("a sequence's length is negative")
        ends = [torch.cat([x.new_zeros(1), x.cumsum(0)]) for x in lens]
        totals = [int(e[-1]) for e in ends]
        cls._sizes(totals[0], totals[-1])
        cls._not_capturing("from_lengths")
        with torch.inference_mode(False):
            on = [e.to(torch.int32).to(device) for e in ends]
        return cls(on[0], on[-1], totals[0], totals[-1], causal, max([int(x.max()) for x in lens if x.numel()], default=0))

    @classmethod
    def from_offsets(cls, q_offsets: torch.Tensor, k_offsets: Optional[torch.Tensor] = None, *, n_q: Optional[int] = None,
                     n_k: Optional[int] = None, causal: bool = False, check: bool = True) -> "PackedSequences":
        """From device offsets ([n_seq + 1], ascending from 0). ``n_q`` and ``n_k``: the rows of the tensors where
        more lie behind the last sequence. With ``check`` the offsets are read back and refused if they do not
        ascend from 0 inside the tensors; without it (graph capture) ``n_q`` must be given (``n_k`` too with
        ``k_offsets``) and bad offsets give wrong results."""
        for x in (q_offsets,) if k_offsets is None else (q_offsets, k_offsets):
            if not isinstance(x, torch.Tensor) or x.dtype not in (torch.int32, torch.int64) or x.dim() != 1 or x.numel() < 1:
                raise ValueError("offsets must be an int32 or int64 tensor [n_seq + 1]")
            if x.device.type != "cuda":
                raise ValueError(f"offsets must be on a HIP device (got {x.device}); the HIP path has no CPU fallback")
            if x.shape != q_offsets.shape or x.device != q_offsets.device:
                raise ValueError("q_offsets and k_offsets must be of the same sequences, on one device")
        sizes, longest = [n_q, n_q if k_offsets is None else n_k], 0
        if k_offsets is None and n_k is not None and n_k != n_q:
            raise ValueError("n_k differs from n_q without k_offsets")
        if check:
            cls._not_capturing("from_offsets with the check")
            for i, x in enumerate((q_offsets, q_offsets if k_offsets is None else k_offsets)):
                host = x.cpu().to(torch.int64)
                if int(host[0]) != 0 or bool((host[1:] < host[:-1]).any()):
                    raise ValueError("offsets must ascend from 0")
                longest = max(longest, int((host[1:] - host[:-1]).max())) if host.numel() > 1 else 0
                if sizes[i] is None:
                    sizes[i] = int(host[-1])
                elif int(host[-1]) > sizes[i]:
                    raise ValueError(f"the last sequence ends at row {int(host[-1])} of {sizes[i]}")
        elif sizes[0] is None or sizes[1] is None:
            raise ValueError("without the check the tensors' rows must be given (n_q, and n_k with k_offsets)")
        cls._sizes(int(sizes[0]), int(sizes[1]))
        with torch.inference_mode(False):
            q = q_offsets.to(torch.int32, copy=True).contiguous()      # a copy: the caller's may change
            k = q if k_offsets is None else k_offsets.to(torch.int32, copy=True).contiguous()
        return cls(q, k, sizes[0], sizes[1], causal, longest)

    @staticmethod
    def _not_capturing(what: str) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} is not for graph capture: build the sequences before it (a flash layer's by a call at "
                               "the same shape), or from device offsets without the check")

    @staticmethod
    def _device(device) -> torch.device:
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"the HIP path takes device tensors (got {device}); it has no CPU fallback")
        return device

    @property
    def device(self) -> torch.device:
        return self.q_offsets.device

    def positions(self) -> torch.Tensor:
        """int32 [n_q]: each query row's place in its sequence, counted from its first key (0 behind the last
        sequence)."""
        self.used()
        return self._positions

    def key_positions(self) -> torch.Tensor:
        """int32 [n_k]: each key's place in its sequence (0 behind the last sequence). Formed anew in each call where the
        keys' sequences are not the rows'."""
        if self.self_attention:
            return self.positions()
        self.used()
        return _op("packed_spans")(self.k_offsets, self.k_offsets, self.n_k, self.n_k, False)[2]


def _check_seqs(seqs, q: torch.Tensor, k: torch.Tensor) -> None:
    if not isinstance(seqs, PackedSequences):
        raise TypeError(f"seqs must be a PackedSequences (got {type(seqs)})")
    if q.size(0) != seqs.n_q or k.size(0) != seqs.n_k:
        raise ValueError(f"the sequences cover ({seqs.n_q} rows, {seqs.n_k} keys), the tensors have ({q.size(0)}, {k.size(0)})")
    if q.device != seqs.device:
        raise ValueError(f"q is on {q.device}, the sequences on {seqs.device}")
    seqs.used()


# ------------------------------------------------------------------ softmax attention
def packed_attention(q, k, v, seqs: PackedSequences, scale: Optional[float] = None, with_lse: bool = False):
    """softmax(scale q k^T) v inside each sequence of a packed batch.

    q [n_q, heads, hn], k and v [n_k, kv_heads, hn] of one dtype (k and v are cast to q's), heads a multiple of
    kv_heads (query head h reads key head h // (heads // kv_heads)), hn a multiple of 8 up to 128. Rows and heads
    may have any strides. ``scale`` (positive, up to 2e38): 1 / sqrt(hn) by default. Returns out [n_q, heads, hn], or (out,
    lse) with ``with_lse``: lse float32 [n_q, heads], the log of the row's sum of exponentials, -inf for a row
    that sees no key (its out is 0); lse is not differentiable. Gradients repeat bit for bit."""
    _check_seqs(seqs, q, k)
    k, v = _as(q, k), _as(q, v)
    scale = 1.0 / math.sqrt(q.size(-1)) if scale is None else float(scale)
    out, lse = _op("packed_attention")(q, k, v, seqs.row_span, seqs.key_span, scale, seqs.longest)
    return (out, lse * math.log(2.0)) if with_lse else out


# ------------------------------------------------------------------ rotary positions
class RotaryFrequencies:
    """The frequencies of rotary positions, formed once on the host in 64 bits.

    Pair i of ``rot`` rotated values turns by theta_i = base^(-2i / rot) radians a position. For contexts longer
    than a model was trained on, ``scaling``:

      "linear"    theta_i / factor
      "ntk"       base * factor^(rot / (rot - 2)) in place of base: fast pairs stay, the slowest is divided by factor
      "by_parts"  pairs that turn at least ``high`` times over ``original`` positions stay, those that turn at
                  most ``low`` times are divided by factor, those between go over linearly in their turns;
                  ``amplitude`` (default 1) scales q and k, as such schemes do with the logits' temperature
    """

    def __init__(self, rot: int, base: float = 10000.0, *, factor: float = 1.0, scaling: str = "linear",
                 original: Optional[int] = None, low: float = 1.0, high: float = 4.0, amplitude: float = 1.0,
                 device="cuda"):
        device = PackedSequences._device(device)
        rot = int(rot)
        if rot < 2 or rot % 2 or rot > 1024:
            raise ValueError(f"rot must be an even number of 2 to 1024 (got {rot})")
        if not (base > 1.0 and math.isfinite(base)) or not (factor > 0.0 and math.isfinite(factor)):
            raise ValueError(f"base {base} must be above 1 and factor {factor} positive")
        if not math.isfinite(amplitude):
            raise ValueError(f"amplitude {amplitude}")
        with torch.inference_mode(False):           # a plain tensor: training saves it
            self.turns = (self._theta(rot, base, factor, scaling, original, low, high) / (2 * math.pi)).to(device)
        self.rot, self.amplitude = rot, float(amplitude)

    @staticmethod
    def _theta(rot, base, factor, scaling, original, low, high) -> torch.Tensor:
        exponent = torch.arange(rot // 2, dtype=torch.float64) * 2 / rot
        if scaling == "linear":
            theta = base ** -exponent / factor
        elif scaling == "ntk":
            if rot < 4:
                raise ValueError("ntk scaling needs two pairs at least")
            theta = (base * factor ** (rot / (rot - 2))) ** -exponent
        elif scaling == "by_parts":
            if original is None or original < 1 or not 0.0 < low < high:
                raise ValueError("by_parts scaling needs original positions and 0 < low < high")
            theta = base ** -exponent
            keep = ((original * theta / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
            theta = theta * keep + theta / factor * (1.0 - keep)
        else:
            raise ValueError(f"scaling {scaling!r} (linear, ntk or by_parts)")
        return theta

    @torch.inference_mode(False)
    def to(self, device) -> "RotaryFrequencies":
        got = object.__new__(RotaryFrequencies)
        got.rot, got.amplitude, got.turns = self.rot, self.amplitude, self.turns.to(PackedSequences._device(device))
        return got


def rotary_embedding(q, k=None, freq: RotaryFrequencies = None, positions: Optional[torch.Tensor] = None,
                     seqs: Optional[PackedSequences] = None, interleaved: bool = False):
    """q (and k) [rows, heads, hn] with the first ``freq.rot`` values of every head turned by the row's position.

    ``positions``: int32 or int64 [rows] on the device, of any size and sign (angles are formed in 64 bits);
    without them each row's place in its sequence: q by ``seqs.positions()``, k by ``seqs.key_positions()`` where it
    has a row for each of the sequences' keys, or as q where it has one for each of their rows (the new tokens' keys,
    before they are put behind the kept ones). Pairs are (i, i + rot / 2), or with
    ``interleaved`` (2i, 2i + 1). Returns new tensors, (q, k) or q alone; gradients are turned back."""
    if not isinstance(freq, RotaryFrequencies):
        raise TypeError(f"freq must be a RotaryFrequencies (got {type(freq)})")
    if positions is None:
        if seqs is None:
            raise ValueError("rotary_embedding needs positions or seqs")
        if seqs.n_q != q.size(0):
            raise ValueError(f"the sequences cover {seqs.n_q} rows, q has {q.size(0)}")
        positions = seqs.positions()
        if k is not None and k.size(0) == seqs.n_k and not seqs.self_attention:      # keys of sequences of their own
            return (rotary_embedding(q, None, freq, positions, interleaved=interleaved),
                    rotary_embedding(_as(q, k), None, freq, seqs.key_positions(), interleaved=interleaved))
    if freq.rot > q.size(-1):
        raise ValueError(f"{freq.rot} rotated values in a head of {q.size(-1)}")
    k = None if k is None else _as(q, k)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    got = _op("rotary_embedding")(q, k, positions, freq.turns, freq.amplitude, bool(interleaved))
    return got[0] if k is None else got


# ------------------------------------------------------------------ linear attention
def _decays(log_decay, q) -> torch.Tensor:
    if not isinstance(log_decay, torch.Tensor) or log_decay.dim() != 1 or log_decay.size(0) != q.size(1):
        raise ValueError(f"log_decay must be [{q.size(1)}]")
    if log_decay.requires_grad:
        raise NotImplementedError("the decays are constants: no gradient with respect to log_decay")
    return log_decay.float().contiguous()


def linear_attention(q, k, v, log_decay, seqs: PackedSequences, scale: Optional[float] = None,
                     initial_state: Optional[torch.Tensor] = None, return_state: bool = False):
    """out_i = scale sum_{j <= i} exp(log_decay (i - j)) (q_i . k_j) v_j inside each sequence: attention without a
    softmax, whose state S_i = exp(log_decay) S_{i-1} + k_i v_i^T has a fixed size.

    q and k [rows, heads, dk], v [rows, heads, dv] of one dtype (k and v are cast to q's), dk and dv multiples of 8
    up to 128; log_decay float32 [heads], at most 0 (0: no decay; -inf: only the row's own token; NaN: the head's results
    are NaN), a constant. A value of v that is not finite makes its column NaN or infinite in the rows that see it, and
    leaves the other columns and rows as they are.
    ``seqs``: causal, the same sequences for rows and keys. ``scale``: 1 / sqrt(dk) by default.
    ``initial_state`` float32 [sequences, heads, dk, dv] comes before each sequence's first token; with
    ``return_state`` (out, state behind the last token) is returned, from which ``linear_attention_step`` or the
    next chunk go on. Gradients flow to q, k and v; the states are constants."""
    _check_seqs(seqs, q, k)
    if not seqs.self_attention or not seqs.causal:
        raise ValueError("linear attention takes causal sequences of the same rows and keys")
    k, v = _as(q, k), _as(q, v)
    if initial_state is not None:
        if initial_state.requires_grad:
            raise NotImplementedError("the initial state is a constant: no gradient with respect to it")
        initial_state = initial_state.float().contiguous()
    scale = 1.0 / math.sqrt(q.size(-1)) if scale is None else float(scale)
    log_decay = _decays(log_decay, q)
    out, state = _op("linear_attention")(q, k, v, log_decay, seqs.row_span, seqs.key_span, seqs.q_offsets, scale,
                                         seqs.longest, initial_state, bool(return_state))
    return (out, state) if return_state else out


def linear_attention_step(q, k, v, log_decay, state, scale: Optional[float] = None,
                          out_state: Optional[torch.Tensor] = None):
    """One token of each of n sequences: (out [n, heads, dv], new state). q and k [n, heads, dk], v [n, heads, dv],
    state float32 [n, heads, dk, dv]. ``out_state``: where the new state is written (``state`` itself updates it in
    place; anything else must not overlap it), else a new tensor. For inference: no gradients."""
    if _trains(q, k, v, state, out_state):
        raise NotImplementedError("linear_attention_step has no gradients (linear_attention has)")
    scale = 1.0 / math.sqrt(q.size(-1)) if scale is None else float(scale)
    return _op("linear_attn_step")(q.contiguous(), _as(q, k).contiguous(), _as(q, v).contiguous(), _decays(log_decay, q), state,
                                   scale, out_state)
