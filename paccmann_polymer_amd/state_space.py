"""Causal convolution and selective state space scan: the operators of a sequence layer beside the StackGRU of K1
(`stack_gru_vae`), for packed batches, for rectangular ones, and for single tokens while generating.  The reference's only sequence
operator is the recurrent one (paccmann_polymer/models/paccmann_encoder.py:166-168); these have no counterpart in it.

Batches.  `x` is a `PackedSequence` (its `.data` [rows, D]), rows [rows, D] of a packed batch with the `plan` that `packed_rows` made of
its batch sizes, or a rectangular tensor [T, B, D] of any strides (a batch-first one goes in as `x.transpose(0, 1)`).  The other
per-step tensors come in the same form.  States [B, ...] are in packed (sorted) order, as K1's `h0` is: permute them with the
PackedSequence's `sorted_indices`.  A program that works on the same packing again keeps the plan: making one copies a few
integers to the device, which cannot be captured into a graph.

Types.  Activations are fp32 or bf16 (all of a call the same); parameters, scan states and their gradients are fp32.  The
convolution's state holds inputs, in their type.  Kernels: csrc/ppk_causal_conv.hip, csrc/ppk_selective_scan.hip.

A backward pass inside a graph capture needs leaves that no eager autograd graph holds at that time (autograd would make the
capturing stream wait for the eager one, which ends the process): take `torch.autograd.grad` of fresh detached leaves, or capture first.
"""
import ctypes
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable
from torch.nn.utils.rnn import PackedSequence

from . import _C

_lib = _C.lib
MAX_TAPS = 8
MAX_STATES = 64
FAR_ROWS = 1 << 30                 # the kernels take rows that are fewer elements apart; others are copied
MAX_ROWS = 1 << 31                 # the kernels count rows in 32 bits


class PackedRows(NamedTuple):
    """What the kernels need of a packed batch; `packed_rows` makes it."""
    offsets: torch.Tensor            # [T + 1] int64, device: step t owns rows offsets[t] .. offsets[t + 1]
    lengths: torch.Tensor            # [B] int64, device
    tiles: torch.Tensor              # [B + 1] int64, device: first kept state of each sequence
    steps: int
    sequences: int
    rows: int
    kept: int                        # kept states in all
    batch_sizes: torch.Tensor        # [T] int64, host: what it was made of


def packed_rows(batch_sizes, device, sequences: Optional[int] = None) -> PackedRows:
    """The plan of a packed batch from its `PackedSequence.batch_sizes` (or the PackedSequence itself).  `sequences`: how many there
    are, where some have no steps at all (they are the last ones, and keep their states)."""
    if isinstance(batch_sizes, PackedSequence):
        batch_sizes = batch_sizes.batch_sizes
    bs = torch.as_tensor(batch_sizes).to('cpu', torch.int64).reshape(-1)
    T = bs.numel()
    B = int(bs[0]) if T else 0
    if T and (int(bs.min()) < 1 or bool((bs[1:] > bs[:-1]).any())):
        raise ValueError('packed_rows: batch sizes must be positive and must not increase')
    if T and int(bs.sum()) >= MAX_ROWS:
        raise ValueError(f'packed_rows: {int(bs.sum())} rows (fewer than 2^31 are supported)')
    if sequences is not None:
        if int(sequences) < B:
            raise ValueError(f'packed_rows: {int(sequences)} sequences, but {B} have a first step')
        B = int(sequences)
    tile = int(_lib.ppk_selective_scan_tile())
    off = torch.zeros(T + 1, dtype=torch.int64)
    off[1:] = torch.cumsum(bs, 0)
    # length of sequence b: how many steps have more than b rows
    lengths = torch.zeros(B, dtype=torch.int64)
    if T:
        lengths[:int(bs[0])] = T - torch.searchsorted(bs.flip(0), torch.arange(int(bs[0])), right=True)
    tiles = torch.zeros(B + 1, dtype=torch.int64)
    tiles[1:] = torch.cumsum((lengths + tile - 1) // tile, 0)
    sent = torch.cat([off, lengths, tiles]).to(device)
    return PackedRows(sent[:T + 1], sent[T + 1:T + 1 + B], sent[T + 1 + B:], T, B, int(off[-1]), int(tiles[-1]), bs)


def _data(t):
    return t.data if isinstance(t, PackedSequence) else t


class _Batch:
    """The layout of a call: packed or rectangular, and how its tensors are addressed."""

    def __init__(self, what, x, plan):
        if isinstance(x, PackedSequence) and plan is None:
            plan = packed_rows(x.batch_sizes, x.data.device)
        data = _data(x)
        if not isinstance(data, torch.Tensor):
            raise TypeError(f'{what}: x must be a tensor or a PackedSequence')
        self.what, self.plan = what, plan
        if plan is not None:
            if not isinstance(plan, PackedRows):
                raise TypeError(f'{what}: plan must be what packed_rows gives')
            if isinstance(x, PackedSequence) and not torch.equal(x.batch_sizes, plan.batch_sizes):
                raise ValueError(f'{what}: the plan is of another packing than x')
            if data.dim() != 2 or data.shape[0] != plan.rows:
                raise ValueError(f'{what}: x must be [{plan.rows}, D] for this plan')
            self.T, self.B, self.rows = plan.steps, plan.sequences, plan.rows
            self.lead, self.out_rows = (plan.rows,), (1, 1)
        else:
            if data.dim() != 3:
                raise ValueError(f'{what}: x must be [T, B, D], or the rows of a packed batch with its plan')
            self.T, self.B, _ = data.shape
            self.rows = self.T * self.B
            self.lead = (self.T, self.B)
            # outputs lie as x does: batch-first where a sequence's steps are next to each other
            self.batch_first = self.T == 1 or data.stride(0) < data.stride(1)
            self.out_rows = (1, self.T) if self.batch_first else (self.B, 1)
        self.D = data.shape[-1]
        if self.D < 1:
            raise ValueError(f'{what}: x has no channels')

    def data_of(self, name, t):
        """The rows of a per-step PackedSequence, which has to be packed as x is."""
        if self.plan is None or not torch.equal(t.batch_sizes, self.plan.batch_sizes):
            raise ValueError(f'{self.what}: {name} is packed in another way than x')
        return t.data

    def take(self, name, t, tail, dtype):
        """A per-step tensor [lead, tail], the elements of its last dimension next to each other."""
        if isinstance(t, PackedSequence):
            t = self.data_of(name, t)
        if not isinstance(t, torch.Tensor) or t.shape != self.lead + tail:
            raise ValueError(f'{self.what}: {name} must be {[*self.lead, *tail]}, not {list(t.shape) if isinstance(t, torch.Tensor) else t}')
        if t.dtype != dtype:
            raise TypeError(f'{self.what}: {name} must be {dtype}, as x is')
        s = t.stride()
        return t if s[0] < FAR_ROWS and s[1] < FAR_ROWS and (s[-1] == 1 or t.shape[-1] == 1) else t.contiguous()

    def strides(self, t):
        """Of a step and of a sequence, in elements; of the only one, whatever the tensor says, 0."""
        if t is None:
            return 0, 0
        s = t.stride()
        if self.plan is not None:
            return (s[0], s[0]) if self.rows > 1 else (0, 0)
        return s[0] if self.T > 1 else 0, s[1] if self.B > 1 else 0

    def new(self, tail, like):
        """An uninitialised per-step tensor of the type and device of `like`, laid out as x is; no view: a caller may change it in place."""
        if self.plan is None and self.batch_first:
            n = tail[0] if len(tail) == 1 else tail[0] * tail[1]
            return like.new_empty_strided(self.lead + tail, (n, self.T * n, *tail[1:], 1))
        return like.new_empty(self.lead + tail)

    def pointers(self):
        p = self.plan
        return (None, None) if p is None else (_C.addr(p.offsets), _C.addr(p.lengths))

    def tensors(self):
        return () if self.plan is None else (self.plan.offsets, self.plan.lengths, self.plan.tiles)


def _param(what, name, t, shape):
    if not isinstance(t, torch.Tensor) or t.shape != shape:
        raise ValueError(f'{what}: {name} must be {list(shape)}')
    if t.dtype != torch.float32:
        raise TypeError(f'{what}: {name} must be float32')


_I64 = {n: ctypes.c_int64 * n for n in (4, 6, 16)}


def _ints(*values):
    return _I64[len(values)](*values)


def _contiguous(t):
    return None if t is None else t.contiguous()


def _ws(nbytes, device):
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def _like(x, y):
    """y in the form that x came in."""
    return PackedSequence(y, x.batch_sizes, x.sorted_indices, x.unsorted_indices) if isinstance(x, PackedSequence) else y


# ------------------------------------------------------------------------------------------------------- causal convolution
class _CausalConv(torch.autograd.Function):

    @staticmethod
    def forward(ctx, batch, silu, x, weight, bias, state):
        dev = x.device
        weight, bias, state = weight.contiguous(), _contiguous(bias), _contiguous(state)
        D, K = weight.shape
        with _C.on_device(dev):
            y = batch.new((D,), x)
            last = x.new_empty((batch.B, K - 1, D))
            off, lengths = batch.pointers()
            _C.check(_lib.ppk_causal_conv_fwd(_C.DTYPES[x.dtype], batch.T, batch.B, D, K, off, lengths, _C.addr(x), _C.addr(weight), _C.addr(bias), _C.addr(state),
                                              silu, _C.addr(y), _C.addr(last), _ints(*batch.strides(x), *batch.strides(y)), _C.stream_on(dev)))
        ctx.save_for_backward(x, weight, bias, state)
        ctx.batch, ctx.silu = batch, silu
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, state = ctx.saved_tensors
        batch, dev = ctx.batch, x.device
        D, K = weight.shape
        with _C.on_device(dev):
            dy = torch.zeros(*batch.lead, D, dtype=x.dtype, device=dev) if dy is None else batch.take('dy', dy, (D,), x.dtype)
            dlast = _contiguous(dlast)
            dx = batch.new((D,), x)
            dw = torch.empty_like(weight)
            db = None if bias is None else torch.empty_like(bias)
            ds = None if state is None else torch.empty_like(state)
            off, lengths = batch.pointers()
            wsb = _lib.ppk_causal_conv_bwd_workspace_bytes(batch.T, batch.B, D, K)
            ws = _ws(wsb, dev)
            _C.check(_lib.ppk_causal_conv_bwd(_C.DTYPES[x.dtype], batch.T, batch.B, D, K, off, lengths, _C.addr(x), _C.addr(weight), _C.addr(bias), _C.addr(state), ctx.silu,
                                              _C.addr(dy), _C.addr(dlast), _C.addr(dx), _C.addr(dw), _C.addr(db), _C.addr(ds),
                                              _ints(*batch.strides(x), *batch.strides(dy), *batch.strides(dx)), _C.addr(ws), wsb, _C.stream_on(dev)))
        return None, None, dx, dw, db, ds


def _conv_params(what, weight, bias, D, activation):
    if not torch.is_tensor(weight) or weight.dim() != 2 or weight.shape[0] != D or weight.shape[1] < 1:
        raise ValueError(f'{what}: weight must be [{D}, taps]')
    if weight.shape[1] > MAX_TAPS:
        raise ValueError(f'{what}: at most {MAX_TAPS} taps')
    _param(what, 'weight', weight, weight.shape)
    if bias is not None:
        _param(what, 'bias', bias, (D,))
    if activation not in (None, 'silu'):
        raise ValueError(f"{what}: activation must be None or 'silu'")
    return int(activation == 'silu')


def causal_conv(x, weight, bias=None, plan: Optional[PackedRows] = None, state=None, activation='silu'):
    """Each channel's causal convolution over its sequence: y_t = act(bias + sum_k weight[:, k] x_{t - K + 1 + k}), and the new state.

    weight [D, K] fp32 (K <= 8, the last tap is the current step's), bias [D] fp32.  state [B, K - 1, D] in x's type: the inputs
    before the first step, the oldest first (None: zeros).  Returns (y like x, new state [B, K - 1, D]: each sequence's last inputs).
    Differentiable in x, weight, bias and state."""
    what = 'causal_conv'
    batch = _Batch(what, x, plan)
    data = _data(x)
    _C.dtype_code(data, what)
    data = batch.take('x', data, (batch.D,), data.dtype)
    silu = _conv_params(what, weight, bias, batch.D, activation)
    K = weight.shape[1]
    if state is not None:
        if not torch.is_tensor(state) or tuple(state.shape) != (batch.B, K - 1, batch.D):
            raise ValueError(f'{what}: state must be {[batch.B, K - 1, batch.D]}')
        if state.dtype != data.dtype:
            raise TypeError(f'{what}: state must be {data.dtype}, as x is')
    _C.one_device(data, weight, bias, state, *batch.tensors())
    y, last = _CausalConv.apply(batch, silu, data, weight, bias, state)
    return _like(x, y), last


def _extent(t):
    """The addresses that a tensor's elements lie between."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a, b):
    """Whether the memory that two tensors span has a part in common."""
    if a is None or b is None or not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    return a0 < b1 and b0 < a1


def _no_gradient(what, **tensors):
    """A step's results are part of no autograd graph: an input that wants a gradient is refused, or it would be lost without a word."""
    for name, t in tensors.items():
        if t is not None and t.requires_grad:
            raise ValueError(f'{what}: {name} requires a gradient (training goes through the form for whole sequences; call this one under torch.no_grad())')


def _step_out(what, state, out, others):
    """Where a step writes its new state: `out`, or fresh memory.  `out` may be the state itself, but share memory with nothing else."""
    if out is None:
        return state.new_empty(state.shape)
    if not torch.is_tensor(out) or out.shape != state.shape or out.dtype != state.dtype or out.device != state.device or not out.is_contiguous():
        raise ValueError(f'{what}: out must be a contiguous tensor like state')
    if out.data_ptr() != state.data_ptr() and _overlap(out, state):
        raise ValueError(f'{what}: out overlaps state without being it')
    for t in others:
        if _overlap(t, out):
            raise ValueError(f'{what}: out shares memory with an input')
    if out.requires_grad:
        raise ValueError(f'{what}: out requires a gradient (training goes through the form for whole sequences)')
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)         # an autograd graph that saved it finds it changed
    return out


def causal_conv_step(x, state, weight, bias=None, activation='silu', out=None):
    """One token of each of B sequences: x [B, D], state [B, K - 1, D] -> (y [B, D], new state).  `out`: where the new state goes
    (it may be `state`: updated in place).  Inference only, an input that wants a gradient is refused: training goes through `causal_conv`."""
    what = 'causal_conv_step'
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f'{what}: x must be [B, D]')
    code = _C.dtype_code(x, what)
    B, D = x.shape
    silu = _conv_params(what, weight, bias, D, activation)
    K = weight.shape[1]
    if not isinstance(state, torch.Tensor) or state.shape != (B, K - 1, D):
        raise ValueError(f'{what}: state must be {[B, K - 1, D]}')
    if state.dtype != x.dtype:
        raise TypeError(f'{what}: state must be {x.dtype}, as x is')
    if torch.is_grad_enabled() and (x.requires_grad or state.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        _no_gradient(what, x=x, state=state, weight=weight, bias=bias)
    dev = _C.one_device(x, state, weight, bias)
    with _C.on_device(dev):
        ld, unit = x.stride()
        if unit != 1 and D != 1:
            x = x.contiguous()
            ld = D
        weight, bias = weight.contiguous(), _contiguous(bias)
        new = _step_out(what, state, out, (x, weight, bias))
        state = state.contiguous()
        y = x.new_empty((B, D))
        _C.check(_lib.ppk_causal_conv_step(code, B, D, K, x.data_ptr(), ld, state.data_ptr(), weight.data_ptr(), _C.addr(bias), silu, y.data_ptr(),
                                           new.data_ptr(), _C.stream_on(dev)))
    return y, new


# ------------------------------------------------------------------------------------------------------------ selective scan
def _scan_strides(batch, x, raw, B, C, z, rows, dy):
    f = batch.strides
    return _ints(*f(x), *f(raw), *f(B), B.stride(-2), *f(C), C.stride(-2), *f(z), *rows, *f(dy))


class _SelectiveScan(torch.autograd.Function):

    @staticmethod
    def forward(ctx, batch, softplus, want_grad, x, dt, A, B, C, D, z, dt_bias, state):
        dev = x.device
        A, D, dt_bias, state = A.contiguous(), _contiguous(D), _contiguous(dt_bias), _contiguous(state)
        N, G, width = A.shape[1], B.shape[-2], batch.D
        tiles = None if batch.plan is None else batch.plan.tiles
        with _C.on_device(dev):
            y = batch.new((width,), x)
            last = A.new_empty((batch.B, width, N))
            kept = None
            if want_grad:
                n = batch.plan.kept if batch.plan is not None else batch.B * -(-batch.T // int(_lib.ppk_selective_scan_tile()))
                kept = A.new_empty((n, width, N))
            off, lengths = batch.pointers()
            wsb = _lib.ppk_selective_scan_fwd_workspace_bytes(batch.T, batch.B, width, N, G)
            ws = _ws(wsb, dev) if wsb else None
            _C.check(_lib.ppk_selective_scan_fwd(_C.DTYPES[x.dtype], batch.T, batch.B, width, N, G, off, lengths, _C.addr(tiles), _C.addr(x), _C.addr(dt), _C.addr(A),
                                                 _C.addr(B), _C.addr(C), _C.addr(D), _C.addr(z), _C.addr(dt_bias), _C.addr(state), softplus, _C.addr(y), _C.addr(last), _C.addr(kept),
                                                 _scan_strides(batch, x, dt, B, C, z, batch.out_rows, None), _C.addr(ws), wsb, _C.stream_on(dev)))
        if kept is not None:
            ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, kept)
            ctx.batch, ctx.softplus, ctx.has_state = batch, softplus, state is not None
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, dt, A, B, C, D, z, dt_bias, kept = ctx.saved_tensors
        batch, dev = ctx.batch, x.device
        N, G, width = A.shape[1], B.shape[-2], batch.D
        tiles = None if batch.plan is None else batch.plan.tiles
        with _C.on_device(dev):
            dy = torch.zeros(*batch.lead, width, dtype=x.dtype, device=dev) if dy is None else batch.take('dy', dy, (width,), x.dtype)
            dlast = _contiguous(dlast)
            dx, draw = batch.new((width,), x), batch.new((width,), x)
            dz = None if z is None else batch.new((width,), x)
            dB, dC = batch.new((G, N), x), batch.new((G, N), x)
            dA = torch.empty_like(A)
            dD = None if D is None else torch.empty_like(D)
            dbias = None if dt_bias is None else torch.empty_like(dt_bias)
            dstate = A.new_empty((batch.B, width, N)) if ctx.has_state else None
            off, lengths = batch.pointers()
            wsb = _lib.ppk_selective_scan_bwd_workspace_bytes(batch.T, batch.B, width, N, G, batch.rows)
            ws = _ws(wsb, dev)
            _C.check(_lib.ppk_selective_scan_bwd(
                _C.DTYPES[x.dtype], batch.T, batch.B, width, N, G, batch.rows, off, lengths, _C.addr(tiles), _C.addr(x), _C.addr(dt), _C.addr(A), _C.addr(B), _C.addr(C),
                _C.addr(D), _C.addr(z), _C.addr(dt_bias), ctx.softplus, _C.addr(kept), _C.addr(dy), _C.addr(dlast), _C.addr(dx), _C.addr(draw), _C.addr(dA), _C.addr(dB), _C.addr(dC),
                _C.addr(dD), _C.addr(dz), _C.addr(dbias), _C.addr(dstate), _scan_strides(batch, x, dt, B, C, z, batch.out_rows, dy), _C.addr(ws), wsb, _C.stream_on(dev)))
        return None, None, None, dx, draw, dA, dB, dC, dD, dz, dbias, dstate


def _scan_params(what, A, D, dt_bias, width):
    if not torch.is_tensor(A) or A.dim() != 2 or A.shape[0] != width or A.shape[1] < 1:
        raise ValueError(f'{what}: A must be [{width}, states]')
    if A.shape[1] > MAX_STATES:
        raise ValueError(f'{what}: at most {MAX_STATES} states a channel')
    _param(what, 'A', A, A.shape)
    if D is not None:
        _param(what, 'D', D, (width,))
    if dt_bias is not None:
        _param(what, 'dt_bias', dt_bias, (width,))
    return A.shape[1]


def _grouped(what, name, t, lead, width, N):
    """B or C as [..., groups, N]."""
    if not isinstance(t, torch.Tensor) or t.dim() not in (len(lead) + 1, len(lead) + 2) or t.shape[-1] != N:
        raise ValueError(f'{what}: {name} must be [..., groups, {N}] or [..., {N}]')
    t = t.unsqueeze(-2) if t.dim() == len(lead) + 1 else t
    if t.shape[-2] < 1 or width % t.shape[-2]:
        raise ValueError(f'{what}: {t.shape[-2]} groups of {width} channels')
    return t


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, plan: Optional[PackedRows] = None, state=None, dt_softplus=True):
    """Selective state space scan: per channel d, with its group's B and C,

      s_t = softplus(dt_t + dt_bias) (or the plain sum);  h_t = exp(s_t A) h_{t-1} + s_t x_t B_t;  y_t = (C_t . h_t + D x_t) silu(z_t)

    x, dt, z [.., channels]; B, C [.., groups, N] or [.., N]; A [channels, N], D, dt_bias [channels] fp32; state [B, channels, N] fp32 (None:
    zeros).  D, z, dt_bias may be None.  Returns (y like x, last state [B, channels, N] fp32).  N <= 64.
    Differentiable in x, dt, A, B, C, D, z, dt_bias and state."""
    what = 'selective_scan'
    batch = _Batch(what, x, plan)
    data, width = _data(x), batch.D
    _C.dtype_code(data, what)
    data = batch.take('x', data, (width,), data.dtype)
    N = _scan_params(what, A, D, dt_bias, width)
    raw = batch.take('dt', dt, (width,), data.dtype)
    gate = None if z is None else batch.take('z', z, (width,), data.dtype)
    B, C = (batch.data_of(n, v) if isinstance(v, PackedSequence) else v for n, v in (('B', B), ('C', C)))
    Bg, Cg = _grouped(what, 'B', B, batch.lead, width, N), _grouped(what, 'C', C, batch.lead, width, N)
    if Bg.shape != Cg.shape:
        raise ValueError(f'{what}: B has {Bg.shape[-2]} groups, C has {Cg.shape[-2]}')
    tail = tuple(Bg.shape[-2:])
    Bg, Cg = batch.take('B', Bg, tail, data.dtype), batch.take('C', Cg, tail, data.dtype)
    if state is not None:
        _param(what, 'state', state, (batch.B, width, N))
    _C.one_device(data, raw, A, Bg, Cg, D, gate, dt_bias, state, *batch.tensors())
    want_grad = torch.is_grad_enabled() and (
        data.requires_grad or raw.requires_grad or A.requires_grad or Bg.requires_grad or Cg.requires_grad or (D is not None and D.requires_grad)
        or (gate is not None and gate.requires_grad) or (dt_bias is not None and dt_bias.requires_grad) or (state is not None and state.requires_grad))
    y, last = _SelectiveScan.apply(batch, int(bool(dt_softplus)), want_grad, data, raw, A, Bg, Cg, D, gate, dt_bias, state)
    return _like(x, y), last


def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, dt_softplus=True, out=None):
    """One token of each of B sequences: x, dt, z [B, channels], B, C [B, groups, N] or [B, N], state [B, channels, N] fp32 -> (y [B, channels],
    new state).  `out`: where the new state goes (it may be `state`: updated in place).  Inference only, an input that wants a gradient is refused:
    training goes through `selective_scan`."""
    what = 'selective_scan_step'
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f'{what}: x must be [B, channels]')
    dtype, code = x.dtype, _C.dtype_code(x, what)
    n, width = x.shape
    N = _scan_params(what, A, D, dt_bias, width)
    B, C = _grouped(what, 'B', B, (n,), width, N), _grouped(what, 'C', C, (n,), width, N)
    if B.shape != C.shape:
        raise ValueError(f'{what}: B has shape {list(B.shape)}, C {list(C.shape)}')
    rows = []
    for name, v, shape in (('x', x, (n, width)), ('dt', dt, (n, width)), ('z', z, (n, width)), ('B', B, (n, *B.shape[1:])), ('C', C, (n, *B.shape[1:]))):
        if v is None and name == 'z':
            rows.append(None)
            continue
        if not isinstance(v, torch.Tensor) or v.shape != shape:
            raise ValueError(f'{what}: {name} must be {list(shape)}')
        if v.dtype != dtype:
            raise TypeError(f'{what}: {name} must be {dtype}, as x is')
        rows.append(v if v.stride(-1) == 1 or shape[-1] == 1 else v.contiguous())
    x, dt, z, B, C = rows
    _param(what, 'state', state, (n, width, N))
    if torch.is_grad_enabled() and (
            x.requires_grad or dt.requires_grad or A.requires_grad or B.requires_grad or C.requires_grad or state.requires_grad or (D is not None and D.requires_grad)
            or (z is not None and z.requires_grad) or (dt_bias is not None and dt_bias.requires_grad)):
        _no_gradient(what, x=x, dt=dt, A=A, B=B, C=C, state=state, D=D, z=z, dt_bias=dt_bias)
    dev = _C.one_device(x, dt, A, B, C, D, z, dt_bias, state)
    with _C.on_device(dev):
        A, D, dt_bias = A.contiguous(), _contiguous(D), _contiguous(dt_bias)
        new = _step_out(what, state, out, (x, dt, A, B, C, D, z, dt_bias))
        state = state.contiguous()
        y = x.new_empty((n, width))
        strides = _ints(0, x.stride(0), 0, dt.stride(0), 0, B.stride(0), B.stride(1), 0, C.stride(0), C.stride(1), 0, 0 if z is None else z.stride(0), 0, 1, 0, 0)
        _C.check(_lib.ppk_selective_scan_step(code, n, width, N, B.shape[1], x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), _C.addr(D),
                                              _C.addr(z), _C.addr(dt_bias), state.data_ptr(), int(bool(dt_softplus)), y.data_ptr(), new.data_ptr(), strides,
                                              _C.stream_on(dev)))
    return y, new
