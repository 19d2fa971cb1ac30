"""Whole-step hipGraph capture for the production trainer.

The training step is ~2k kernel launches (backbone fwd/bwd + prototype
ops + Adam + EM); at MI355X speeds launch overhead is a measurable slice
of the 45 ms step. ``GraphedStep`` captures the ENTIRE step — forward,
losses, backward, optimizer.step and the (inline) EM update — into one
hipGraph and replays it per batch, copying the batch into static input
buffers. The same recipe bench.py has always measured; this module makes
it the path ``train.py`` actually runs (the
reference's driver and bench were one program, reference main.py:234-287).

Capture constraints and how they are met:

* no eager autograd graph of the same parameters is alive — steps stay
  eager while one is;
* static shapes — replay only when the incoming batch is full-size;
  remainder batches fall back to the eager path (the caller checks
  ``matches()``);
* optimizer state must exist before capture — the first ``warmup_steps``
  calls run eagerly on a side stream (they are REAL training steps);
* Adam must be constructed with ``capturable=True`` (train.py does when
  graphs are enabled);
* phase flips (warm<->joint optimizer swap, mining on, EM on), other loss
  weights, another learning rate or ``clip_grad_norm``, and
  ``use_mx4``/``no_mx4`` change the captured program — the step signature is checked per call and the graph is
  re-captured when it changes (a handful of times per run);
* the EM update runs INLINE in the graph (no side stream: cross-stream
  event sync inside capture is legal but buys nothing when every step
  runs EM);
* the library's memset nodes (weight gradients of convolutions, reductions)
  become fill kernels before the graph is instantiated: such nodes write
  wrongly in later replays on this hardware (utils/graphs.py);
* per-step scalars (loss terms, batch accuracy) are written into static
  device buffers inside the graph and read by the trainer afterwards —
  no host sync is added.

Multi-rank: RCCL collectives are capturable in principle but unvalidated
on an 8-GPU node; graphs stay single-rank unless MGPROTO_GRAPH_DIST=1
(same gate as bench.py).
"""

import os
from typing import Optional

import torch
import torch.nn.functional as F

from ..models.conv1x1 import GemmConv2d
from ..utils.graphs import capture_graph, eager_graph_of


def graphs_enabled(device, world: int = 1) -> bool:
    if device is None or device.type != 'cuda':
        return False
    if os.environ.get('MGPROTO_NO_GRAPH') == '1':
        return False
    return world == 1 or os.environ.get('MGPROTO_GRAPH_DIST') == '1'


class GraphedStep:
    """Captured (or capture-pending) training step.

    Usage from the trainer loop::

        gs = GraphedStep(model, aux, coefs, device, batch, img, amp_dtype)
        ...
        if gs.matches(image, optimizer, use_mine, em_active):
            stats = gs.step(image, target, optimizer, reducer, em_active,
                            use_mine)
        else:
            ...eager path...

    ``stats`` is a dict of DEVICE scalars: loss / ce / mine / aux /
    n_correct / grad_norm (floats accumulate trainer-side exactly like the eager
    path's detached tensors).
    """

    def __init__(self, model, aux_criterion, coefs, device, batch_size,
                 img_size, amp_dtype='bf16', warmup_steps=3,
                 channels_last=True, clip_grad_norm=None):
        self.model = model
        self.aux = aux_criterion
        self.coefs = coefs
        self.device = device
        self.batch_size = batch_size
        self.warmup_steps = warmup_steps
        self.amp_dtype = amp_dtype
        self.clip_grad_norm = clip_grad_norm
        self.graph: Optional[torch.cuda.CUDAGraph] = None
        self.broken = False          # capture failed -> permanent eager
        self._sig = None
        self._warm_count = 0
        self._said = False

        self.static_img = torch.zeros(batch_size, 3, img_size, img_size,
                                      device=device)
        if channels_last:
            self.static_img = self.static_img.to(
                memory_format=torch.channels_last)
        self.static_tgt = torch.zeros(batch_size, dtype=torch.int64,
                                      device=device)
        z = lambda: torch.zeros((), device=device)  # noqa: E731
        self.stats = {'loss': z(), 'ce': z(), 'mine': z(), 'aux': z(),
                      'n_correct': z(), 'grad_norm': z()}

    # ------------------------------------------------------------------
    def _signature(self, optimizer, use_mine, em_active):
        return (id(optimizer), bool(use_mine), bool(em_active),
                self.clip_grad_norm,
                # numbers are part of the program, tensors are read by it
                tuple(sorted((k, v) for k, v in self.coefs.items())),
                tuple((k, v) for g in optimizer.param_groups
                      for k, v in g.items()
                      if isinstance(v, (bool, int, float, tuple))),
                tuple(p.requires_grad for p in self.model.parameters()),
                tuple(m.mx4 for m in self.model.modules()
                      if isinstance(m, GemmConv2d)))

    def matches(self, image, optimizer, use_mine, em_active) -> bool:
        """Can this batch go through the graphed path (possibly after a
        (re)capture)?"""
        if self.broken:
            return False
        if image.shape[0] != self.batch_size:
            return False
        sig = self._signature(optimizer, use_mine, em_active)
        if sig != self._sig:
            # program changed: drop the old graph, restart warmup
            self._sig = sig
            self.graph = None
            self._warm_count = 0
        return True

    # ------------------------------------------------------------------
    def _compute(self, optimizer, reducer, em_active, use_mine):
        """One full training step on the static buffers. Runs eagerly
        during warmup/capture; replayed thereafter."""
        with torch.autocast(device_type='cuda',
                            dtype=torch.bfloat16 if self.amp_dtype == 'bf16'
                            else torch.float16,
                            enabled=self.amp_dtype in ('bf16', 'fp16')):
            output, x_aux = self.model(self.static_img, self.static_tgt)
        output = output.float()
        if use_mine and output.shape[2] > 1:
            mine_loss = sum(F.cross_entropy(output[:, :, k], self.static_tgt)
                            for k in range(1, output.shape[2])) \
                / (output.shape[2] - 1)
        else:
            mine_loss = torch.zeros((), device=self.device)
        ce = F.cross_entropy(output[:, :, 0], self.static_tgt)
        aux_loss = (self.aux(x_aux.float(), self.static_tgt)
                    if self.aux is not None
                    else torch.zeros((), device=self.device))
        loss = (self.coefs['crs_ent'] * ce + self.coefs['mine'] * mine_loss
                + self.coefs['aux'] * aux_loss)

        if reducer is not None:
            reducer.prepare()
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        if reducer is not None:
            reducer.finalize()
        if self.clip_grad_norm is not None:
            from .trainer import clip_optimizer_grads
            self.stats['grad_norm'].copy_(
                clip_optimizer_grads(optimizer, self.clip_grad_norm))
        optimizer.step()
        if em_active:
            self.model.update_GMM()

        pred = torch.argmax(output[:, :, 0].detach(), dim=1)
        self.stats['loss'].copy_(loss.detach())
        self.stats['ce'].copy_(ce.detach())
        self.stats['mine'].copy_(mine_loss.detach())
        self.stats['aux'].copy_(aux_loss.detach())
        self.stats['n_correct'].copy_(
            (pred == self.static_tgt).sum().to(self.stats['n_correct'].dtype))

    # ------------------------------------------------------------------
    def step(self, image, target, optimizer, reducer=None, em_active=False,
             use_mine=False) -> dict:
        """Run one training step on this batch (eager warmup -> capture ->
        replay). Call only after ``matches()`` returned True."""
        self.static_img.copy_(image, non_blocking=True)
        self.static_tgt.copy_(target, non_blocking=True)

        if self.graph is None:
            wait = self._warm_count >= self.warmup_steps and eager_graph_of(
                [*self.model.parameters(), *(p for g in optimizer.param_groups
                                             for p in g['params'])])
            if wait and not self._said:
                self._said = True
                print('# hipGraph capture waits: an eager autograd graph of '
                      'these parameters is alive (a loss or output that '
                      'someone keeps)', flush=True)
            if wait or self._warm_count < self.warmup_steps:
                # real training steps, staged on a side stream so the
                # allocations warm the capture pool
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    self._compute(optimizer, reducer, em_active, use_mine)
                torch.cuda.current_stream().wait_stream(side)
                self._warm_count += 1
                return self.stats
            try:
                self.graph, _ = capture_graph(
                    lambda: self._compute(optimizer, reducer, em_active,
                                          use_mine))
                # the capture itself did not execute: replay once so THIS
                # batch trains too
                self.graph.replay()
            except Exception as e:  # noqa: BLE001
                print(f'# hipGraph capture failed ({type(e).__name__}: {e});'
                      ' continuing eager', flush=True)
                self.broken = True
                self._compute(optimizer, reducer, em_active, use_mine)
            return self.stats

        self.graph.replay()
        return self.stats
