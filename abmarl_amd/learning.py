"""The policy operators (include/gw_learn.h): from a policy's logits to the
engine's action rows, and from a rollout's slabs to the policy's gradient.

    r = sample_actions(logits, heads, noise)        # action rows, log-probabilities
    out = engine.rollout(...)                       # slabs [K][E][A]
    adv = advantages(out['reward'], value, out['done'], marks, live)
    loss = policy_loss(logits, r.actions, adv.advantage, r.logp, heads, valid=adv.valid)
    cut = fragment_cuts(marks, steps)               # where its memory starts anew
    h, last = linear_recurrence(gate, x, state, cut=cut[:-1])   # a policy's memory, x [K][E]...

GridWorldEngine has sample_actions, advantages, policy_loss, policy_loss_grad and
linear_recurrence as methods that fill in its own heads, lanes, marks and cuts.  Tensors stay on the GPU and the calls only put work on the
current stream of the tensors' device: they can be captured into a graph.
Wrong arguments raise ValueError before anything is launched.  Like the
engine, the operators have no CPU fallback.
"""
import ctypes as C
from collections import namedtuple

import torch
from torch.autograd import forward_ad

from abmarl_amd import _native

MARK_END, MARK_TRUNCATED, MARK_RESET, MARK_SKIP = 1, 2, 4, 8
SEGMENT = 16                       # GW_RECURRENCE_SEGMENT
MAX_HEADS = 256                    # GW_MAX_HEADS

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

Sampled = namedtuple('Sampled', 'actions logp entropy')
PolicyLoss = namedtuple('PolicyLoss', 'loss stats count logp')
PolicyGradient = namedtuple('PolicyGradient', 'loss stats count logp grad')
Advantages = namedtuple('Advantages', 'advantage target valid')


class _Heads(C.Structure):
    """gw_policy_heads"""
    _fields_ = [('n_heads', C.c_int32), ('act_dim', C.c_int32), ('sizes', C.POINTER(C.c_int32)),
                ('low', C.POINTER(C.c_int32)), ('slots', C.POINTER(C.c_int32))]


class PolicyHeads:
    """The softmax heads of a policy over action rows: head d chooses among
    sizes[d] values low[d], low[d] + 1, ... of action column slots[d].  A row
    of logits holds the heads side by side (n_choices values); an action row
    has act_dim ints, those that no head has are 0.  By default the heads are
    the columns, and their values start at 0."""

    def __init__(self, sizes, low=None, slots=None, act_dim=None):
        self.sizes = tuple(int(v) for v in sizes)
        n = len(self.sizes)
        self.low = tuple(int(v) for v in low) if low is not None else (0,) * n
        self.slots = tuple(int(v) for v in slots) if slots is not None else tuple(range(n))
        self.act_dim = int(act_dim) if act_dim is not None else max(self.slots, default=0) + 1
        _need(1 <= n <= MAX_HEADS, f"{n} heads: 1 to {MAX_HEADS}")
        _need(len(self.low) == n and len(self.slots) == n, "sizes, low and slots are one value per head")
        _need(min(self.sizes) >= 1, f"head sizes {self.sizes}: at least one choice each")
        _need(len(set(self.slots)) == n and 0 <= min(self.slots) and max(self.slots) < self.act_dim <= 32767,
              f"slots {self.slots}: different columns of an action row of {self.act_dim}")
        self.n_heads, self.n_choices = n, sum(self.sizes)
        _need(self.n_choices <= 1 << 30, f"{self.n_choices} choices: at most 2^30")
        _need(all(-2**31 <= v and v + s <= 2**31 for v, s in zip(self.low, self.sizes)), "action values exceed int32")
        ints = C.c_int32 * n
        self._c = _Heads(n, self.act_dim, ints(*self.sizes), ints(*self.low), ints(*self.slots))
        self._p = C.addressof(self._c)

    def __repr__(self):
        return f"PolicyHeads(sizes={self.sizes}, low={self.low}, slots={self.slots}, act_dim={self.act_dim})"


# ------------------------------------------------------------------- checks
def _need(cond, message):
    if not cond:
        raise ValueError(message)


def _at(t):
    return None if t is None else t.data_ptr()


def _tensor(t, name, dtypes, device=None, shape=None):
    """t is a contiguous tensor of one of the dtypes, there, of that shape
    (this runs in every call: messages are made only for errors)."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: a tensor is needed, not {type(t).__name__}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: {t.dtype}, not one of {', '.join(str(d) for d in dtypes)}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, not {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, not on {device}")
    return t


_INF = float('inf')
_FLOATS = tuple(_DTYPES)
_BYTES = (torch.uint8, torch.bool)
_F32 = (torch.float32,)
_I32 = (torch.int32,)


def _rows(t, name, width):
    """(rows, elements between rows) of a matrix of logits: the last dimension
    side by side, the others one stride."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: a tensor is needed, not {type(t).__name__}")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name}: {t.dtype}, not float32, float16 or bfloat16")
    if t.dim() < 1 or t.shape[-1] != width:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, not (..., {width})")
    if t.is_contiguous():
        return t.numel() // width, width
    _need(t.stride(-1) == 1 or width == 1, f"{name}: the choices of a row must lie side by side")
    rows, ld = 1, None
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if ld is None:
            ld = stride
        _need(stride == ld * rows, f"{name}: the rows must lie one stride apart (strides {t.stride()})")
        rows *= size
    ld = width if ld is None else ld
    _need(ld >= width or t.numel() == 0, f"{name}: rows of {width} must not overlap (strides {t.stride()})")
    return t.numel() // width, ld


def _mask(t, shape, device):
    """(mask or None, mask rows): choice_mask has the trailing dimensions of the logits."""
    if t is None:
        return None, 0
    k = t.dim() if isinstance(t, torch.Tensor) else -1
    if not (1 <= k <= len(shape) and t.shape == shape[len(shape) - k:] or
            k == 2 and len(shape) == 2 and t.shape[1] == shape[1] and t.shape[0] >= 1 and shape[0] % t.shape[0] == 0):
        raise ValueError(f"choice_mask: shape {tuple(t.shape) if k >= 0 else type(t).__name__} is not that of the "
                         f"logits' last dimensions {tuple(shape)}")
    _tensor(t, 'choice_mask', _BYTES, device)
    return t, t.numel() // shape[-1]


def _gpu(device):
    if device.type != 'cuda':
        raise RuntimeError("the policy operators need a ROCm GPU (no CPU fallback).")


_libs = None


def _lib():
    global _libs
    if _libs is None:
        _libs = _native.learn_lib()
    return _libs


_device_now, _stream_of = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _call(fn, device, *args):
    """fn(*args, stream) with the tensors' device the current one, on that
    device's current stream."""
    i = device.index
    if _device_now() == i:
        st = fn(*args, _stream_of(i))
    else:
        with torch.cuda.device(i):
            st = fn(*args, _stream_of(i))
    if st:
        _native.check_learn(st, fn.__name__)


def _once():
    # (autograd runs a backward pass with gradients off unless it is to be
    # differentiated itself)
    if torch.is_grad_enabled():
        raise RuntimeError("the policy operators' gradients cannot be differentiated again (create_graph)")


def _no_tangent(*inputs):
    # (kernels read values only: a tangent would be lost without a word)
    if forward_ad._current_level >= 0 and any(
            isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in inputs):
        raise NotImplementedError("the policy operators have no forward-mode derivatives")


# ------------------------------------------------------------------ sampling
def sample_actions(logits, heads, noise=None, choice_mask=None, out=None):
    """Draws an action row for each row of logits [..., n_choices] (float32,
    float16 or bfloat16).

    noise: float32 like the logits; with Gumbel noise, -log(Exponential(1)),
    the choices follow the softmax.  None: the likeliest choice of each head.
    The choice is the largest float(logit) + noise, the lowest of equals.
    choice_mask: uint8 or bool with the logits' last dimensions (one row for
    all, one per lane, or one per row): 0 for choices that there are not.  A
    logit of -inf is none either.  A head without any choice gives its first
    value, log-probability 0 and entropy 0.
    out: int32 [..., act_dim] to write the actions to (engine.actions).

    Returns (actions int32 [..., act_dim], logp float32 [...], entropy
    float32 [...]); logp sums the chosen log-probabilities over the heads,
    entropy the heads' entropies.  No gradient flows through them."""
    n, ld = _rows(logits, 'logits', heads.n_choices)
    device, lead = logits.device, logits.shape[:-1]
    if noise is not None:
        _tensor(noise, 'noise', _F32, device, logits.shape)
    mask, mask_rows = _mask(choice_mask, logits.shape, device)
    if out is not None:
        _tensor(out, 'out', _I32, device, lead + (heads.act_dim,))
    _gpu(device)
    if out is None:
        out = torch.empty(lead + (heads.act_dim,), dtype=torch.int32, device=device)
    logp = torch.empty(lead, dtype=torch.float32, device=device)
    entropy = torch.empty(lead, dtype=torch.float32, device=device)
    _call(_lib().gw_policy_sample, device, heads._p, _DTYPES[logits.dtype], n, logits.data_ptr(), ld, _at(noise),
          _at(mask), mask_rows, out.data_ptr(), logp.data_ptr(), entropy.data_ptr())
    return Sampled(out, logp, entropy)


# ---------------------------------------------------------------------- loss
def _loss_args(logits, actions, advantage, old_logp, heads, ref_logits, valid, choice_mask, clip, denominator):
    """The checked arguments that forward and backward share."""
    n, ld = _rows(logits, 'logits', heads.n_choices)
    device, lead = logits.device, logits.shape[:-1]
    ld_ref = 0
    if ref_logits is not None:
        _, ld_ref = _rows(ref_logits, 'ref_logits', heads.n_choices)
        if ref_logits.shape != logits.shape or ref_logits.dtype != logits.dtype or ref_logits.device != device:
            raise ValueError("ref_logits: shape, dtype and device must be the logits'")
    _tensor(actions, 'actions', _I32, device, lead + (heads.act_dim,))
    _tensor(advantage, 'advantage', _F32, device, lead)
    _tensor(old_logp, 'old_logp', _F32, device, lead)
    if valid is not None:
        _tensor(valid, 'valid', _BYTES, device, lead)
    mask, mask_rows = _mask(choice_mask, logits.shape, device)
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    low, high = float(low), float(high)
    if not (0 <= low and C.c_float(low).value < _INF and 0 <= high and C.c_float(high).value < _INF):
        raise ValueError(f"clip {clip}: finite in float32, not negative")
    value, at = 0.0, None
    if isinstance(denominator, torch.Tensor):
        at = _tensor(denominator, 'denominator', _F32, device, torch.Size([]))
    elif denominator is not None:
        value = C.c_float(float(denominator)).value
        _need(0 < value < _INF, f"denominator {denominator}: finite and positive in float32")
    if advantage.requires_grad or old_logp.requires_grad or ref_logits is not None and ref_logits.requires_grad:
        raise ValueError("advantage, old_logp, ref_logits: no gradient flows to them, detach them")
    return n, ld, ld_ref, mask, mask_rows, low, high, value, at


def _finite(name, v):
    v = float(v)
    if not abs(C.c_float(v).value) < _INF:               # (as the kernels take it)
        raise ValueError(f"{name} {v}: must be finite in float32")
    return v


def _launch_loss(logits, actions, advantage, old_logp, ref, valid, heads, args, kl_coef, entropy_coef,
                 grad_scale=1.0, upstream=None, loss=None, stats=None, logp=None, grad=None, denominator_at=None):
    n, ld, ld_ref, mask, mask_rows, low, high, value, at = args
    L, device = _lib(), logits.device
    size = L.gw_policy_loss_workspace(n)
    work = torch.empty(size, dtype=torch.uint8, device=device)
    _call(L.gw_policy_loss, device, heads._p, _DTYPES[logits.dtype], n, logits.data_ptr(), ld, _at(ref), ld_ref,
          actions.data_ptr(), advantage.data_ptr(), old_logp.data_ptr(), _at(valid), _at(mask), mask_rows, low, high,
          kl_coef, entropy_coef, value, _at(at if denominator_at is None else denominator_at), grad_scale,
          _at(upstream), _at(loss), _at(stats), _at(logp), _at(grad), work.data_ptr(), size)


def _loss_outputs(logits):
    device = logits.device
    return (torch.empty((), dtype=torch.float32, device=device), torch.empty(5, dtype=torch.float32, device=device),
            torch.empty(logits.shape[:-1], dtype=torch.float32, device=device))


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, advantage, old_logp, ref, valid, mask, at, heads, args, kl_coef, entropy_coef):
        loss, stats, logp = _loss_outputs(logits)
        _launch_loss(logits, actions, advantage, old_logp, ref, valid, heads, args, kl_coef, entropy_coef,
                     loss=loss, stats=stats, logp=logp)
        ctx.save_for_backward(logits, actions, advantage, old_logp, ref, valid, mask, at, stats)
        ctx.rest = heads, args, kl_coef, entropy_coef
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(stats, logp)
        return loss, stats, logp

    @staticmethod
    def backward(ctx, d_loss, _stats, _logp):
        _once()
        logits, actions, advantage, old_logp, ref, valid, mask, at, stats = ctx.saved_tensors
        heads, args, kl_coef, entropy_coef = ctx.rest
        if d_loss is None:
            return (None,) * 12
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        _launch_loss(logits, actions, advantage, old_logp, ref, valid, heads, args, kl_coef, entropy_coef,
                     upstream=d_loss.contiguous(), grad=grad, denominator_at=stats[4])
        return (grad,) + (None,) * 11


def policy_loss(logits, actions, advantage, old_logp, heads, *, ref_logits=None, valid=None, choice_mask=None,
                clip=0.2, kl_coef=0.0, entropy_coef=0.0, denominator=None):
    """The clipped policy loss with a KL and an entropy term, differentiable by
    the logits.  Over the valid rows,

        loss = mean(-min(ratio A, clamp(ratio, 1 - clip, 1 + clip) A)
                    + kl_coef KL(softmax(ref) || softmax(logits)) - entropy_coef H(softmax(logits)))

    with ratio = exp(logp - old_logp) and logp the log-probability of the
    row's action, summed over the heads, as are KL and H.

    logits, ref_logits: [..., n_choices] float32, float16 or bfloat16, rows one stride
    apart; ref_logits None: no KL.  actions: int32 [..., act_dim] as
    sample_actions gives them.  advantage, old_logp: float32 [...].  valid: uint8 or
    bool [...]: rows with 0 (agents that did not act) count for nothing, whatever
    stands in them, and get no gradient.  choice_mask: as sample_actions'.  clip: one number, or the lower
    and the upper.  denominator: what to divide by instead of the number of
    valid rows (a number or a float32 device scalar, e.g. all ranks' rows).
    An action whose choice there is not has probability 0: logp -inf, ratio 0.

    Returns (loss, stats, count, logp): the means of the policy term, the KL,
    the entropy and of the clipped rows in stats float32 [4], the denominator
    in count, logp float32 [...] (0 for rows not valid); only loss has a gradient.
    The sums over rows are double and their order is fixed: equal inputs give equal bits."""
    args = _loss_args(logits, actions, advantage, old_logp, heads, ref_logits, valid, choice_mask, clip, denominator)
    kl_coef, entropy_coef = _finite('kl_coef', kl_coef), _finite('entropy_coef', entropy_coef)
    _gpu(logits.device)
    loss, stats, logp = _PolicyLoss.apply(logits, actions, advantage, old_logp, ref_logits, valid, args[3], args[8],
                                          heads, args, kl_coef, entropy_coef)
    return PolicyLoss(loss, stats[:4], stats[4], logp)


def policy_loss_grad(logits, actions, advantage, old_logp, heads, *, ref_logits=None, valid=None, choice_mask=None,
                     clip=0.2, kl_coef=0.0, entropy_coef=0.0, denominator=None, grad_scale=1.0):
    """policy_loss and its gradient by the logits in one pass over them:
    (loss, stats, count, logp, grad), grad like the logits, times grad_scale
    (the loss scale of fp16 training).  For `logits.backward(grad)`; one pass
    reads the logits once where policy_loss and its backward read them twice."""
    args = _loss_args(logits, actions, advantage, old_logp, heads, ref_logits, valid, choice_mask, clip, denominator)
    kl_coef, entropy_coef = _finite('kl_coef', kl_coef), _finite('entropy_coef', entropy_coef)
    grad_scale = _finite('grad_scale', grad_scale)
    _no_tangent(logits, advantage, old_logp, ref_logits)
    device = logits.device
    _gpu(device)
    loss, stats, logp = _loss_outputs(logits)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=device)
    _launch_loss(logits, actions, advantage, old_logp, ref_logits, valid, heads, args, kl_coef, entropy_coef,
                 grad_scale=grad_scale, loss=loss, stats=stats, logp=logp, grad=grad)
    return PolicyGradient(loss, stats[:4], stats[4], logp, grad)


# ---------------------------------------------------------------- recurrence
def _span(shape, t, name):
    """How many channels of x [T, ...] one value of t [T, ...] stands for."""
    if t.shape == shape:
        return 1
    k = t.dim()
    lead = t.shape[:-1] if k == len(shape) and t.shape[-1] == 1 else t.shape
    if not (1 <= len(lead) <= len(shape) and lead == shape[:len(lead)]):
        raise ValueError(f"{name}: shape {tuple(t.shape)} is neither x's {tuple(shape)} nor the first dimensions of it")
    n = 1
    for s in shape[len(lead):]:
        n *= s
    return max(n, 1)                       # (no channels: nothing is read)


def _launch_recurrence(gate, value, gate_span, x, state, cut, cut_span, reverse, h, last, carry):
    T = x.shape[0]
    n = x.numel() // T if T else last.numel()
    L, device = _lib(), x.device
    size = L.gw_recurrence_workspace(T, n)
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _call(L.gw_recurrence, device, _DTYPES[x.dtype], _DTYPES[x.dtype if gate is None else gate.dtype], T, n,
          x.data_ptr(), _at(gate), gate_span, value, _at(cut), cut_span, _at(state), reverse, h.data_ptr(),
          last.data_ptr(), _at(carry), _at(work), size)


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, state, cut, value, gate_span, cut_span, reverse):
        T = x.shape[0]
        h = torch.empty_like(x)
        last = torch.empty(x.shape[1:], dtype=torch.float32, device=x.device)
        carry = torch.empty((-(-T // SEGMENT), last.numel()), dtype=torch.float32, device=x.device)
        _launch_recurrence(gate, value, gate_span, x, state, cut, cut_span, reverse, h, last, carry)
        ctx.save_for_backward(gate, x, cut, carry)
        ctx.rest = value, gate_span, cut_span, reverse, state is not None
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    def backward(ctx, dh, dlast):
        _once()
        gate, x, cut, carry = ctx.saved_tensors
        value, gate_span, cut_span, reverse, has_state = ctx.rest
        if dh is None and dlast is None:
            return (None,) * 8
        T, device = x.shape[0], x.device
        n = carry.shape[1]
        dx = torch.empty_like(x)
        # (without channels no launch writes the gradient of the gates that they would share)
        dgate = (torch.empty_like(gate) if n else torch.zeros_like(gate)) \
            if gate is not None and ctx.needs_input_grad[0] else None
        dstate = torch.empty(x.shape[1:], dtype=torch.float32, device=device) \
            if has_state and ctx.needs_input_grad[2] else None
        dh = None if dh is None else dh.contiguous()
        dlast = None if dlast is None else dlast.contiguous()
        L = _lib()
        size = L.gw_recurrence_backward_workspace(T, n, gate_span)
        work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        _call(L.gw_recurrence_backward, device, _DTYPES[x.dtype], _DTYPES[x.dtype if gate is None else gate.dtype], T, n,
              x.data_ptr(), _at(gate), gate_span, value, _at(cut), cut_span, carry.data_ptr(), reverse, _at(dh),
              _at(dlast), dx.data_ptr(), _at(dgate), _at(dstate), _at(work), size)
        return dgate, dx, dstate, None, None, None, None, None


def linear_recurrence(gate, x, state=None, cut=None, reverse=False):
    """h[t] = gate[t] h[t-1] + x[t] over the first dimension of x [T, ...]
    (float32, float16 or bfloat16), from h[-1] = state (float32 [...], None:
    zeros); with reverse h[t] = gate[t] h[t+1] + x[t] from state behind the
    last step.  Returns (h like x, last float32 [...]: h after the last step
    done).  Sums and states are held in float32.

    gate: like x, or x's first dimensions (channels share a gate; a last
    dimension of 1 may stand for them), of x's dtype or float32; or one number.
    cut: uint8 or bool, x's first dimensions: where it is not 0 the state is
    dropped before the step, as at the first step of an episode (fragment_cuts
    makes it of a rollout's marks, which stand at an episode's last step; a gate
    of 0 drops the state too, whatever it holds).

    Differentiable by gate, x and state (backwards only); a shared gate's gradient
    is summed in a fixed order.  One step (T = 1) is the form for acting."""
    if not isinstance(x, torch.Tensor) or x.dim() < 2:
        raise ValueError("x: a tensor [steps, ...] is needed")
    _tensor(x, 'x', _FLOATS)
    shape, device = x.shape, x.device
    value, gate_span = 0.0, 1
    if isinstance(gate, torch.Tensor):
        _tensor(gate, 'gate', (x.dtype, torch.float32), device)
        gate_span = _span(shape, gate, 'gate')
    else:
        value, gate = _finite('gate', gate), None
    if state is not None:
        _tensor(state, 'state', _F32, device, shape[1:])
    cut_span = 1
    if cut is not None:
        _tensor(cut, 'cut', _BYTES, device)
        cut_span = _span(shape, cut, 'cut')
    reverse = int(bool(reverse))
    _no_tangent(gate, x, state)
    _gpu(device)
    if torch.is_grad_enabled() and (x.requires_grad or (gate is not None and gate.requires_grad) or
                                    (state is not None and state.requires_grad)):
        return _Recurrence.apply(gate, x, state, cut, value, gate_span, cut_span, reverse)
    h = torch.empty_like(x)
    last = torch.empty(shape[1:], dtype=torch.float32, device=device)
    _launch_recurrence(gate, value, gate_span, x, state, cut, cut_span, reverse, h, last, None)
    return h, last


# ---------------------------------------------------------------- advantages
def fragment_marks(all_done, steps=None, horizon=0, autoreset='next_step', all_done_before=None, err=None):
    """What each step of a rollout was to its env: uint8 [K, E] of MARK_END (the
    episode ended with it), MARK_TRUNCATED (the horizon ended it), MARK_RESET
    (no step: the env was reset) and MARK_SKIP (the env raised somewhere in
    the fragment, its rows are not all written).

    all_done: the rollout's uint8 [K, E] slab; all_done_before uint8 [E] and
    steps int32 [E]: the '__all__' and the envs' step counters before it
    (engine.fragment_start()); err int32 [E]: the engine's flags after it, if
    they were 0 before it.  With 'same_step' the observation
    behind a horizon is the next episode's: such a step is marked MARK_END."""
    _tensor(all_done, 'all_done', _BYTES)
    _need(all_done.dim() == 2, f"all_done: shape {tuple(all_done.shape)}, not (steps, envs)")
    K, E = all_done.shape
    device = all_done.device
    if steps is not None:
        _tensor(steps, 'steps', _I32, device, torch.Size([E]))
    if all_done_before is not None:
        _tensor(all_done_before, 'all_done_before', _BYTES, device, torch.Size([E]))
    if err is not None:
        _tensor(err, 'err', _I32, device, torch.Size([E]))
    _need(autoreset in ('same_step', 'next_step'), f"autoreset {autoreset!r}: 'same_step' or 'next_step'")
    _need(0 <= int(horizon) < 2**31, f"horizon {horizon}")
    _gpu(device)
    marks = torch.empty((K, E), dtype=torch.uint8, device=device)
    _call(_lib().gw_fragment_marks, device, K, E, all_done.data_ptr(), _at(all_done_before), _at(steps), _at(err),
          int(horizon), 1 if autoreset == 'same_step' else 2, marks.data_ptr())
    return marks


def fragment_cuts(marks, steps=None):
    """Where a policy's memory starts anew in a rollout: uint8 [K + 1, E] for the
    observations before each step and after the last, linear_recurrence's cut for
    x [K + 1, E, ...] (or cut[:K] for x [K, E, ...]).

    marks: fragment_marks' [K, E].  An observation is an episode's first where the
    step before it ended one (same_step) or was the reset (next_step).  The memory
    of an episode that the horizon ended still reaches the observation behind
    it, whose value advantages() uses; behind an END the reset's own row, which
    nothing uses, stands alone.  steps: int32 [E], the envs' step counters before
    the fragment (engine.fragment_start()): 0 where its first observation is an
    episode's first; None: the state given goes on everywhere."""
    _tensor(marks, 'marks', (torch.uint8,))
    _need(marks.dim() == 2, f"marks: shape {tuple(marks.shape)}, not (steps, envs)")
    K, E = marks.shape
    if steps is not None:
        _tensor(steps, 'steps', _I32, marks.device, torch.Size([E]))
    cut = torch.zeros((K + 1, E), dtype=torch.uint8, device=marks.device)
    cut[1:] = (marks & (MARK_END | MARK_RESET)) != 0
    if steps is not None:
        cut[0] = steps == 0
    return cut


def advantages(reward, value, done, marks, live, gamma=0.99, lam=0.95, acts=None):
    """Generalized advantages and value targets over a rollout's slabs.

    reward: float64 or float32 [K, E, A]; value: float32, float16 or bfloat16
    [K + 1, E, A], of the observations before each step and after the last;
    done: uint8 [K, E, A]; marks: fragment_marks' [K, E]; live: uint8 or bool [E, A],
    lanes not done before the first step; acts: uint8 or bool [A], lanes that act at all.

    For steps in which a lane acted
        delta = reward + gamma value[t+1] - value[t]
        advantage = delta + gamma lam advantage[t+1],  target = advantage + value[t]
    without value[t+1] where the lane or its episode is done, without
    advantage[t+1] there and where the horizon ended it.  Others are 0.
    Returns (advantage, target float32, valid uint8), all [K, E, A]; sums are
    held in float32.  No gradient flows through them."""
    _tensor(reward, 'reward', (torch.float64, torch.float32))
    _need(reward.dim() == 3, f"reward: shape {tuple(reward.shape)}, not (steps, envs, lanes)")
    K, E, A = shape = reward.shape
    device = reward.device
    _tensor(value, 'value', _FLOATS, device, torch.Size([K + 1, E, A]))
    _tensor(done, 'done', _BYTES, device, shape)
    _tensor(marks, 'marks', (torch.uint8,), device, torch.Size([K, E]))
    _tensor(live, 'live', _BYTES, device, torch.Size([E, A]))
    if acts is not None:
        _tensor(acts, 'acts', _BYTES, device, torch.Size([A]))
    gamma, lam = _finite('gamma', gamma), _finite('lam', lam)
    _gpu(device)
    adv = torch.empty(shape, dtype=torch.float32, device=device)
    target = torch.empty(shape, dtype=torch.float32, device=device)
    valid = torch.empty(shape, dtype=torch.uint8, device=device)
    L = _lib()
    size = L.gw_recurrence_workspace(K, E * A)
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _call(L.gw_advantages, device, _DTYPES[value.dtype], int(reward.dtype == torch.float64), K, E, A, reward.data_ptr(),
          value.data_ptr(), done.data_ptr(), marks.data_ptr(), live.data_ptr(), _at(acts), gamma, lam, adv.data_ptr(),
          target.data_ptr(), valid.data_ptr(), _at(work), size)
    return Advantages(adv, target, valid)
