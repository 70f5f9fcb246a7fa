"""clip_grad_norm_ + SGD(momentum, weight_decay) fused over the model's flat arenas
(reference tools/train_ssl_uem.py:169-170,228-232: torch.optim.SGD + clip_grad.clip_grad_norm_(32))."""
import torch

from . import _lib, ops
from .ops import UemError, call, ptr, stream


def _arena_of(params):
    """the model whose flat gradient arena IS the gradients of `params`: all of them are its parameters, each has its slot of the arena as its
    gradient (not None, as behind torch's zero_grad(set_to_none=True), whose slots hold what an earlier pass left, and no tensor of the
    caller's), and none that it trains or that has a gradient is missing (frozen ones may be, as in
    `filter(lambda p: p.requires_grad, model.parameters())`).  Else None"""
    owner = getattr(params[0], "_uem_owner", None) if params else None
    if owner is None or any(getattr(p, "_uem_owner", None) is not owner for p in params):
        return None
    listed = {id(p) for p in params}
    if not all(id(p) in listed or not (p.requires_grad or p.grad is not None) for p in owner.parameters()):
        return None
    base = owner.flat_parameters()[1].data_ptr()
    attached = (p.grad is not None and p.grad.data_ptr() == base + 4 * p._uem_off or not p.requires_grad and p.grad is None for p in params)
    return owner if all(attached) else None


def _holds_sums(model):
    """does the model's gradient arena hold sums over ranks (DataParallel.reduce_gradients), whose average FusedSGD.step would take?"""
    summed = getattr(model, "_uem_summed", None)
    return summed is not None and any(p.grad is summed for p in model.parameters())


def grad_norm(model):
    """L2 norm of the flat gradient arena -> 1-element device tensor (two-stage deterministic reduce)."""
    arena, garena, n = model.flat_parameters()
    partial = torch.empty(_lib.UEM_NORM_BLOCKS, device=arena.device, dtype=torch.float32)
    norm = torch.empty(1, device=arena.device, dtype=torch.float32)
    call("uem_grad_sqnorm", ptr(garena), n, ptr(partial), ptr(norm), stream())
    return norm


def _norm_kind(norm_type, what):
    kind = {2.0: 2, float("inf"): 0}.get(float(norm_type))
    if kind is None:
        raise UemError(f"{what}: norm_type must be 2 or inf, got {norm_type}")
    return kind


def _tensors(given, what):
    """a tensor or an iterable of them, as a list"""
    given = [given] if isinstance(given, torch.Tensor) else list(given)
    for t in given:
        if not isinstance(t, torch.Tensor):
            raise UemError(f"{what}: expected tensors, got {type(t).__name__}")
    return given


def _finite(norm, what):
    if not bool(torch.isfinite(norm)):
        raise UemError(f"{what}: the total norm is {float(norm)}, so nothing is scaled (error_if_nonfinite=False would let it through)")


def get_total_norm(tensors, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """The norm over all elements of all `tensors` (a tensor or an iterable; fp32 and bf16 may be mixed), as a 0-dim fp32 device tensor:
    torch.nn.utils.get_total_norm for norm_type 2 or inf.  Squares are summed in 64 bits, in a fixed order.  error_if_nonfinite reads the norm on
    the host and raises where it is infinite or none (otherwise no value is read there); `foreach` chooses nothing: there is one way."""
    what = "get_total_norm"
    ops.grad_join()                # gradients of arena parameters among them may still be on the side / second stream
    norm = _lib.host().multi_norm(_tensors(tensors, what), what, _norm_kind(norm_type, what), False, None)
    norm = torch.tensor(0.0) if norm is None else norm
    if error_if_nonfinite:
        _finite(norm, what)
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2, error_if_nonfinite=False, foreach=None):
    """Drop-in for torch.nn.utils.clip_grad_norm_: scales the gradients of `parameters` (a tensor or an iterable) in place by
    min(max_norm / (norm + 1e-6), 1) and returns their total norm, a device scalar; norm_type is 2 or inf.  error_if_nonfinite reads the norm
    on the host and raises, with nothing scaled, where it is infinite or none; `foreach` chooses nothing: there is one way.

    ALL trained parameters of one uemda_amd model: its flat gradient arena is clipped in one pass.  Any other list -- some of a model's
    parameters, modules outside a model arena, a model together with other modules, fp32 and bf16 mixed -- is clipped tensor by tensor in
    two passes over the list, and nothing beside it; parameters without a gradient are skipped, gradients that share memory are refused.

    Behind `DataParallel.reduce_gradients` a model's gradients are SUMS over the ranks (FusedSGD.step takes `max_norm` and the average in one
    pass), other modules' are whatever the caller made of them: a list of both is refused."""
    what = "clip_grad_norm_"
    params = _tensors(parameters, what)
    kind, max_norm = _norm_kind(norm_type, what), float(max_norm)
    if not max_norm >= 0.0:
        raise UemError(f"{what}: max_norm must not be negative, got {max_norm}")
    model = _arena_of(params) if kind == 2 else None
    ops.grad_join()                # weight gradients still on the side / second stream (a backward that raised never ran its join callback)
    if model is None:
        owners = {id(o): o for o in (getattr(p, "_uem_owner", None) for p in params if not p.is_leaf or p.grad is not None)}
        if len(owners) > 1 and any(o is not None and _holds_sums(o) for o in owners.values()):
            raise UemError(f"{what}: the list mixes a model's gradients, which are sums over ranks since reduce_gradients(), with others: clip the "
                           "model by FusedSGD.step(max_norm=..., grad_prescale=...) and the others by themselves, once they are reduced and averaged")
        if error_if_nonfinite:
            norm = _lib.host().multi_norm(params, what, kind, True, None)
            if norm is not None:
                _finite(norm, what)
        norm = _lib.host().multi_norm(params, what, kind, True, max_norm)
        return torch.zeros((), device=params[0].device if params else "cpu") if norm is None else norm
    arena, garena, n = model.flat_parameters()
    norm = grad_norm(model)
    if error_if_nonfinite:
        _finite(norm, what)
    coef = torch.clamp(max_norm / (norm + 1e-6), max=1.0)      # one scalar
    call("uem_scale_by_scalar", ptr(garena), None, n, ptr(coef), stream())
    return norm[0]


class FusedSGD(torch.optim.Optimizer):
    """torch.optim.SGD(lr, momentum, weight_decay) semantics (no nesterov / dampening) in ONE pass over
    the flat parameter arena; `step(max_norm=...)` also fuses clip_grad_norm_ into that pass."""

    def __init__(self, model, lr=1e-2, momentum=0.9, weight_decay=5e-4):
        self.model = model
        super().__init__(list(model.parameters()), dict(lr=lr, momentum=momentum, weight_decay=weight_decay))
        arena, _, _ = model.flat_parameters()
        self.momentum_buffer = torch.zeros_like(arena)
        self._steps = 0
        self.last_grad_norm = None

    def zero_grad(self, set_to_none=False):
        self.model.zero_grad()

    def _trainable_ranges(self, n):
        """[(offset, count)] runs of the flat arena that belong to trainable parameters: the whole arena unless something is frozen."""
        params = self.param_groups[0]["params"]
        if all(p.requires_grad for p in params):
            return [(0, n)]
        runs = []
        for p in params:
            if not p.requires_grad:
                continue
            off, cnt = p._uem_off, p.numel()
            if runs and runs[-1][0] + runs[-1][1] == off:
                runs[-1] = (runs[-1][0], runs[-1][1] + cnt)
            else:
                runs.append((off, cnt))
        return runs

    # learning rate as a device scalar (None: by value from param_groups): set by uemda_amd.step.GraphedStep, whose captured
    # optimizer launch would otherwise keep the learning rate of the capture
    lr_device = None

    @torch.no_grad()
    def step(self, closure=None, max_norm=None, grad_prescale=1.0):
        g = self.param_groups[0]
        arena, garena, n = self.model.flat_parameters()
        ops.grad_join()            # no-op after a clean backward (its end-of-backward callback joined); the safety net after one that raised
        norm = None
        if max_norm is not None:
            norm = grad_norm(self.model)
            self.last_grad_norm = norm
        for off, cnt in self._trainable_ranges(n):
            # frozen parameters (requires_grad False: ResNetEncoder freeze_at / batchnorm_trainable) are skipped altogether, as
            # torch.optim.SGD skips a parameter whose .grad is None -- no weight decay, no momentum
            call("uem_sgd_clip_step", ptr(arena) + 4 * off, ptr(garena) + 4 * off, ptr(self.momentum_buffer) + 4 * off, cnt, ptr(norm),
                 float(max_norm) if max_norm is not None else 0.0, float(g["lr"]), float(g["momentum"]),
                 float(g["weight_decay"]), 1 if self._steps == 0 else 0, float(grad_prescale), ptr(self.lr_device), stream())
        self._steps += 1
        if grad_prescale != 1.0:
            self.model._uem_summed = None      # the kernel has left the average in the arena
        ops.weights_changed()
