"""PreconditioningConfig, the template step of every preconditioned gradient maker and the update cadences
(field names, defaults and behaviour of asdl/precondition/prec_grad_maker.py:22-254)."""
import math
import warnings
from dataclasses import dataclass
from typing import Any, List

import torch.nn as nn

from .clipping import clip_grad_norm_
from .grad_maker import GradientMaker
from .profiling import nvtx_range, phase_mark

__all__ = ['PreconditionedGradientMaker', 'PreconditioningConfig', 'get_update_schedule',
           'INTERVAL_CONSTANT', 'INTERVAL_STEP', 'INTERVAL_LINEAR', 'INTERVAL_TYPES']

INTERVAL_CONSTANT = 'constant'
INTERVAL_STEP = 'step'
INTERVAL_LINEAR = 'linear'
INTERVAL_TYPES = [INTERVAL_CONSTANT, INTERVAL_STEP, INTERVAL_LINEAR]

_default_interval = 1
_invalid_value = -1


@dataclass
class PreconditioningConfig:
    """Configuration of gradient preconditioning.

    ``ema_decay`` is the weight of the NEW statistic:
    ``curv_ema = curv_ema * (1 - ema_decay) + curv_new * ema_decay``; -1 disables the moving average.
    ``ignore_modules``: modules, module classes or (parts of) module names to leave alone.
    ``max_grad_norm``: the gradients of all parameters, as they are when the step ends, are scaled down to this 2-norm as one vector
    (None: not); the norm before is the maker's ``grad_norm``."""
    num_total_steps: int = None
    preconditioner_upd_interval: int = _default_interval
    preconditioner_warmup_steps: int = 0
    preconditioner_upd_ratio: float = 1.
    preconditioner_warmup_ratio: float = 0.
    preconditioner_interval_type: str = INTERVAL_CONSTANT
    curvature_upd_interval: int = None
    curvature_warmup_steps: int = 0
    curvature_upd_ratio: float = None
    curvature_warmup_ratio: float = 0.
    curvature_interval_type = INTERVAL_CONSTANT
    data_size: int = _invalid_value
    damping: float = 1.e-7
    ema_decay: float = _invalid_value
    ignore_modules: List[Any] = None
    max_grad_norm: float = None


class _Cadence:
    """When an update is due: a per-step list of booleans (num_total_steps given) or every `interval` steps after
    `warmup` steps of updating every step."""

    def __init__(self, flags=None, interval=1, warmup=0, horizon=None):
        self.flags, self.interval, self.warmup, self.horizon = flags, interval, warmup, horizon

    def due(self, step: int) -> bool:
        if self.flags is None:
            return step < self.warmup or (step - self.warmup) % self.interval == 0
        try:
            return self.flags[step]
        except IndexError:
            warnings.warn(f'Step {step} lies outside the {self.horizon} steps of num_total_steps: no update.')
            return False


class PreconditionedGradientMaker(GradientMaker):
    """Template of one preconditioned step (asdl/precondition/prec_grad_maker.py:68-201):

        [forward + backward]  ->  [update_curvature]  ->  [update_preconditioner]  ->  precondition

    Subclasses fill in the four stages and say through do_forward_and_backward() whether the plain passes run.
    The curvature follows the preconditioner's cadence unless it has an interval or a ratio of its own.  Modules
    are kept in `module_dict` under their names with '/' for '.', leaves with trainable parameters only."""
    _supported_classes = None

    def __init__(self, model: nn.Module, config: PreconditioningConfig):
        super().__init__(model)
        self.config = config
        self._preconditioner_cadence, self._curvature_cadence = self._cadences(config)
        self.state = dict(step=0)
        self.grad_norm = None
        kept = {}
        for name, module in model.named_modules():
            if self._is_supported(name, module):
                kept[name.replace('.', '/')] = module
        self.module_dict = nn.ModuleDict(kept)
        self.device = next(self.module_dict.parameters()).device

    @staticmethod
    def _cadences(config):
        """(preconditioner, curvature) cadences; the second is None when the curvature follows the first."""
        total = config.num_total_steps
        if total is None:
            precond = _Cadence(interval=config.preconditioner_upd_interval, warmup=config.preconditioner_warmup_steps)
            curv = None
            if config.curvature_upd_interval is not None:
                curv = _Cadence(interval=config.curvature_upd_interval, warmup=config.curvature_warmup_steps)
            return precond, curv
        # a known horizon: the ratios decide, the intervals are not looked at
        if config.preconditioner_upd_interval != _default_interval:
            warnings.warn('num_total_steps is set: preconditioner_upd_ratio decides, preconditioner_upd_interval is '
                          'not used.')
        precond = _Cadence(get_update_schedule(total, config.preconditioner_upd_ratio,
                                               config.preconditioner_warmup_ratio), horizon=total)
        curv = None
        if config.curvature_upd_ratio is not None:
            if config.curvature_upd_interval is not None:
                warnings.warn('num_total_steps is set: curvature_upd_ratio decides, curvature_upd_interval is not '
                              'used.')
            curv = _Cadence(get_update_schedule(total, config.curvature_upd_ratio, config.curvature_warmup_ratio),
                            horizon=total)
        elif config.curvature_upd_interval is not None:
            curv = _Cadence(interval=config.curvature_upd_interval, warmup=config.curvature_warmup_steps)
        return precond, curv

    # plain attributes in the reference (asdl/precondition/prec_grad_maker.py:85-99): a user may assign a list of
    # booleans, which then decides like a schedule derived from num_total_steps, or None
    @property
    def preconditioner_upd_schedule(self):
        return self._preconditioner_cadence.flags

    @preconditioner_upd_schedule.setter
    def preconditioner_upd_schedule(self, flags):
        self._preconditioner_cadence.flags = flags
        self._preconditioner_cadence.horizon = None if flags is None else len(flags)

    @property
    def curvature_upd_schedule(self):
        return None if self._curvature_cadence is None else self._curvature_cadence.flags

    @curvature_upd_schedule.setter
    def curvature_upd_schedule(self, flags):
        if self._curvature_cadence is None:
            if flags is None:
                return
            config = self.config
            interval = config.curvature_upd_interval if config.curvature_upd_interval is not None \
                else config.preconditioner_upd_interval
            self._curvature_cadence = _Cadence(interval=interval, warmup=config.curvature_warmup_steps)
        self._curvature_cadence.flags = flags
        self._curvature_cadence.horizon = None if flags is None else len(flags)
        if flags is None and self.config.curvature_upd_interval is None and self.config.curvature_upd_ratio is None:
            self._curvature_cadence = None          # the curvature follows the preconditioner again

    def _is_ignored(self, module_name: str, module: nn.Module) -> bool:
        """config.ignore_modules lists module objects, module classes and substrings of module names."""
        for entry in self.config.ignore_modules or ():
            if isinstance(entry, type):
                hit = isinstance(module, entry)
            elif isinstance(entry, str):
                hit = entry in module_name
            else:
                hit = entry is module
            if hit:
                return True
        return False

    def _is_supported(self, module_name: str, module: nn.Module) -> bool:
        is_leaf = next(module.children(), None) is None
        trainable = any(p.requires_grad for p in module.parameters())
        if not is_leaf or not trainable or self._is_ignored(module_name, module):
            return False
        if self._supported_classes is None or isinstance(module, self._supported_classes):
            return True
        warnings.warn(f'{type(self).__name__} has no curvature for {module} ({module_name}): it is left to the plain '
                      'gradient.')
        return False

    def state_dict(self) -> dict:
        return self.state

    def load_state_dict(self, state_dict: dict):
        self.state['step'] = state_dict['step']

    def forward_and_backward(self):
        step = self.state['step']
        self._startup()
        run_passes = self.do_forward_and_backward(step)
        # (range / phase name, stage, does it run this step?); the names are the phase keywords of the reference's
        # profiling example (examples/prof/README.md:24).  The questions are asked when their stage's turn comes.
        stages = (('fwd', self.forward, lambda: run_passes),
                  ('bwd', self.backward, lambda: run_passes),
                  ('upd_curv', self.update_curvature, lambda: self.do_update_curvature(step)),
                  ('upd_inv', self.update_preconditioner, lambda: self.do_update_preconditioner(step)),
                  ('precond', self.precondition, lambda: True),
                  ('clip', self.clip_gradients, lambda: self.config.max_grad_norm is not None))
        for name, stage, wanted in stages:
            if wanted():
                with nvtx_range(name):
                    stage()
                phase_mark(name)
        self._teardown()
        self.state['step'] += 1
        return self._model_output, self._loss

    # ---- stages (subclasses)
    def _startup(self):
        pass

    def update_curvature(self):
        pass

    def update_preconditioner(self):
        pass

    def precondition(self):
        raise NotImplementedError

    def clip_gradients(self):
        """Scales all gradients of the model down to config.max_grad_norm; their norm before is kept, on the device."""
        self.grad_norm = clip_grad_norm_(self.model.parameters(), self.config.max_grad_norm)

    def _teardown(self):
        pass

    def do_forward_and_backward(self, step=None) -> bool:
        raise NotImplementedError

    # ---- cadence queries (step=None: the current step)
    def do_update_preconditioner(self, step=None) -> bool:
        return self._preconditioner_cadence.due(self.state['step'] if step is None else step)

    def do_update_curvature(self, step=None) -> bool:
        cadence = self._curvature_cadence or self._preconditioner_cadence
        return cadence.due(self.state['step'] if step is None else step)


def get_update_schedule(num_total_steps: int, update_ratio: float = 1., warmup_ratio: float = 0.,
                        interval_type: str = INTERVAL_CONSTANT, reverse=False):
    """One boolean per step: True where an update happens (asdl/precondition/prec_grad_maker.py:204-254).

    int(num_total_steps * update_ratio) updates in all.  The first int(num_total_steps * warmup_ratio) steps all
    update; the remaining updates are laid over the remaining steps
      'constant': every floor(steps / updates)-th step, starting with the first,
      'step':     back to back at the start,
      'linear':   with gaps of 0, D, 2D, ... steps between them, D = floor(2 (steps - n) / (n (n - 1))) for
                  n + 1 updates (n < 2 divides by zero, as in the reference).
    reverse=True returns the list back to front."""
    def in_unit_interval(name, value):
        if not 0 <= value <= 1:
            raise ValueError(f'{name} = {value} is outside [0, 1].')

    if num_total_steps <= 0:
        raise ValueError(f'num_total_steps = {num_total_steps} has to be positive.')
    in_unit_interval('update_ratio', update_ratio)
    in_unit_interval('warmup_ratio', warmup_ratio)
    updates = int(num_total_steps * update_ratio)
    warmup = int(num_total_steps * warmup_ratio)
    if warmup > updates:
        raise ValueError(f'{warmup} warm-up steps need more than the {updates} updates that update_ratio allows.')
    if interval_type not in INTERVAL_TYPES:
        raise ValueError(f'interval_type {interval_type!r} is not one of {INTERVAL_TYPES}.')

    steps_left, updates_left = num_total_steps - warmup, updates - warmup
    positions = list(range(warmup))                     # steps that update
    if updates_left > 0:
        if interval_type == INTERVAL_CONSTANT:
            stride = steps_left // updates_left
            positions += [warmup + j * stride for j in range(updates_left)]
        elif interval_type == INTERVAL_STEP:
            positions += [warmup + j for j in range(updates_left)]
        else:
            n = updates_left - 1
            growth = math.floor(2 * (steps_left - n) / n / (n - 1))
            at = warmup
            positions.append(at)
            for i in range(n):
                at += growth * i + 1
                positions.append(at)
    if positions and positions[-1] >= num_total_steps:
        raise ValueError(f'The {interval_type} layout of {updates} updates ends at step {positions[-1] + 1} > '
                         f'num_total_steps = {num_total_steps}.')
    flags = [False] * num_total_steps
    for at in positions:
        flags[at] = True
    return flags[::-1] if reverse else flags
