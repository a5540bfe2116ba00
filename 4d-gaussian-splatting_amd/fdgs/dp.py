"""View-parallel data parallelism: one process per GPU, replicas of the
Gaussians / grids / MLP, each rank renders its own views.

The reference has no distributed code; its trainer already loops over a list of
views and averages one loss over them (src/runner/fdgs_trainer.py:239-248,
127-130), and that loop is the seam used here.  One exchange step per
iteration: a single flat-bucket SUM all-reduce of every parameter gradient
(RCCL over xGMI when the backend is "nccl"), plus three small reductions of the
densification statistics the trainer keeps (fdgs_trainer.py:125-126,146-148):
radii MAX, visibility MAX (= OR), summed view-space gradient SUM.
"""
import contextlib
import os

import torch
import torch.distributed as dist

# RCCL's all-reduce: the ring algorithm.  The gradients are tens of megabytes and xGMI is point to point, which is what a
# ring is for.  Must be set before the communicator is created; a value the user has set is left alone.
os.environ.setdefault("NCCL_ALGO", "Ring")

# FDGS_DP_SINGLE_RANK=1: take the exchange step even in a group of one rank (a rehearsal of the RCCL calls on a
# one-GPU machine; the reductions are then identities)
_SINGLE_RANK = os.environ.get("FDGS_DP_SINGLE_RANK") == "1"


_LOCAL_ONLY = False


@contextlib.contextmanager
def local_only():
    """Inside the block this rank behaves as a group of its own: every view of a batch stays here and no exchange
    step is taken.  For timing the same batch on ONE GPU from inside an N-rank job (the other ranks must not step
    meanwhile: the replicas differ afterwards)."""
    global _LOCAL_ONLY
    before, _LOCAL_ONLY = _LOCAL_ONLY, True
    try:
        yield
    finally:
        _LOCAL_ONLY = before


def is_dist():
    return (not _LOCAL_ONLY and dist.is_available() and dist.is_initialized()
            and (dist.get_world_size() > 1 or _SINGLE_RANK))


def rank_world():
    if not _LOCAL_ONLY and dist.is_available() and dist.is_initialized():
        return dist.get_rank(), dist.get_world_size()
    return 0, 1


def all_reduce_(t, op, group=None):
    """In-place all-reduce.  RCCL ("nccl") takes device tensors as they are; with the gloo backend (CPU
    rehearsals of the exchange step) a device tensor is staged through host memory here, explicitly."""
    if t.is_cuda and dist.get_backend(group) == "gloo":
        h = t.cpu()
        dist.all_reduce(h, op=op, group=group)
        t.copy_(h)
    else:
        dist.all_reduce(t, op=op, group=group)


class _Completed:
    """Handle of a reduction that has already taken place."""

    def wait(self):
        return True


def all_reduce_async(t, op=None, group=None):
    """Starts an in-place SUM all-reduce of `t` on the communication stream and returns a handle; its wait()
    orders the current stream after the collective without blocking the host, so kernels enqueued between
    the two calls run beside it.  Always returns a handle: with gloo staging of a device tensor the reduction is
    complete on return and the handle's wait() does nothing (callers take "no handle" to mean "no collective")."""
    op = dist.ReduceOp.SUM if op is None else op
    if t.is_cuda and dist.get_backend(group) == "gloo":
        all_reduce_(t, op, group)
        return _Completed()
    return dist.all_reduce(t, op=op, group=group, async_op=True)


@torch.no_grad()
def broadcast_parameters(params, src=0, group=None):
    """Makes every rank's replica bit-identical to rank `src`'s (one flat broadcast)."""
    params = list(params)
    if not is_dist() or not params:
        return
    flat = torch.cat([p.detach().reshape(-1).to(torch.float32) for p in params])
    if flat.is_cuda and dist.get_backend(group) == "gloo":
        h = flat.cpu()
        dist.broadcast(h, src=src, group=group)
        flat.copy_(h)
    else:
        dist.broadcast(flat, src=src, group=group)
    torch._foreach_copy_([p.data for p in params], [v.view_as(p) for p, v in
                                                     zip(params, flat.split_with_sizes([p.numel() for p in params]))])


def shard_views(views, rank=None, world=None):
    """Rank r takes views r, r+W, r+2W, ... of the global batch."""
    if rank is None:
        rank, world = rank_world()
    return list(views[rank::world])


def local_loss_scale(n_local, n_global):
    """The reference's loss is a mean over the concatenated batch
    (src/model/losses.py:7-8 via fdgs_trainer.py:495): each rank sums its
    per-view means scaled by 1/B_global, and the SUM all-reduce of the
    gradients reproduces the gradient of the global mean."""
    del n_local
    return 1.0 / float(n_global)


class GradBucket:
    """Flat fp32 bucket over a fixed parameter list: one collective per step."""

    def __init__(self, params):
        self.params = [p for p in params if p.requires_grad]
        self.numel = sum(p.numel() for p in self.params)
        self.flat = None

    def rebuild(self, params):
        """After densification / pruning changed N."""
        self.__init__(params)

    def allreduce_(self, group=None):
        """SUM all-reduce of every .grad that exists, written back in place.  A tensor without a gradient stays
        without one (the optimizer then skips it and does not count a step for it, as torch.optim.Adam does for
        the deformation field during the coarse stage).  Which tensors have gradients must be the same on every
        rank: it follows from the stage, and a rank without views fills in zeros for that same set."""
        have = [p for p in self.params if p.grad is not None]
        if not have:
            return
        sizes = [p.numel() for p in have]
        total = sum(sizes)
        dev = have[0].device
        if self.flat is None or self.flat.numel() < total or self.flat.device != dev:
            self.flat = torch.empty(max(total, self.numel), device=dev, dtype=torch.float32)
        flat = self.flat[:total]
        # gather and scatter with one concatenation and one multi-tensor copy (not a launch pair per tensor)
        torch.cat([p.grad.reshape(-1) for p in have], out=flat)
        if is_dist():
            all_reduce_(flat, dist.ReduceOp.SUM, group)
        torch._foreach_copy_([p.grad for p in have], [v.view_as(p) for p, v in zip(have, flat.split_with_sizes(sizes))])


def reduce_densification_stats(radii, visibility, viewspace_grad, group=None):
    """radii [N] int32 -> MAX, visibility [N] bool -> OR, viewspace_grad [N,3] -> SUM (sum, then norm,
    as fdgs_trainer.py:146-148 + gaussian_model.py:183)."""
    if not is_dist():
        return radii, visibility, viewspace_grad
    r = radii.contiguous()
    all_reduce_(r, dist.ReduceOp.MAX, group)
    if visibility is not None:          # None: the caller derives it as radii > 0, which commutes with the MAX
        v = visibility.to(torch.uint8).contiguous()
        all_reduce_(v, dist.ReduceOp.MAX, group)
        visibility = v.bool()
    g = viewspace_grad
    if g is not None:                   # None: the caller has summed it with the parameter gradients
        g = g.contiguous()
        all_reduce_(g, dist.ReduceOp.SUM, group)
    return r, visibility, g
