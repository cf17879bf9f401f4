"""The distillation term of the joint step: a mean over the RoIs that the NMS kept, on all ranks.  The zero
boxes that fill an image's rows up take no part."""
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from objectdetection_amd.train import FRCNModel, TrainStep
from test_train_step import CFG, OraclePathOps, _data, _free_port, _grads, _models

T, KEPT = 2.0, (17, 5, 24)


class Ops(OraclePathOps):
    """Image i keeps KEPT[i] RoIs; the distillation as torch operations."""

    def targets(self, fmap, pred_reg, pred_obj, gt, label, seed, image_base):
        t = super().targets(fmap, pred_reg, pred_obj, gt, label, seed, image_base)
        kept = torch.tensor(KEPT[image_base:image_base + gt.shape[0]])
        t["roi_weight"] = (torch.arange(CFG.post_n) < kept[:, None]).float()
        return t

    def distill_loss(self, logits, top_values, top_index, temperature, weight=None):
        p = torch.softmax(top_values / temperature, -1)
        log_q = torch.log_softmax(logits / temperature, -1).gather(-1, top_index)
        loss = temperature ** 2 * (p * (torch.log(p) - log_q)).sum(-1)
        self.rows = loss.detach()
        return loss.mean() if weight is None else (loss * weight).sum() / weight.sum().clamp(min=1.0)


class Teacher(torch.nn.Module):
    """Logits that differ from RoI to RoI, image `first` and the following ones'."""

    def __init__(self, first):
        super().__init__()
        self.first = first

    def logits(self, pooled):
        B, R = pooled.shape[:2]
        table = 3 * torch.randn((3, R, CFG.num_classes), generator=torch.Generator().manual_seed(8))
        return None, table[self.first:self.first + B]


def step_of(world, rank=0, d=None, ops=None):
    rpn, frcn = _models()
    teacher = Teacher(rank)
    return TrainStep(rpn, frcn, CFG, ops or Ops(CFG), d, rank, world, teacher=teacher, distill_temperature=T,
                     distill_weight=3.0, bucket_bytes=64 << 10)


def test_the_mean_is_over_the_kept_rois():
    step = step_of(1)
    images, gt, label = _data(3)
    losses = step.forward_backward(images, gt, label, seed=4)
    rows = step.ops.rows
    want = 3.0 * torch.cat([rows[i, :n] for i, n in enumerate(KEPT)]).mean()
    assert abs(float(losses[4]) - float(want)) <= 1e-5 * float(want)
    assert abs(float(losses[4]) - 3.0 * float(rows.mean())) > 1e-3 * float(want)


def test_path_operations_without_weights_average_all_rows():
    class Plain(Ops):
        def targets(self, *a):
            t = super().targets(*a)
            del t["roi_weight"]
            return t

        def distill_loss(self, logits, top_values, top_index, temperature):
            return super().distill_loss(logits, top_values, top_index, temperature)

    step = step_of(1, ops=Plain(CFG))
    images, gt, label = _data(2)
    losses = step.forward_backward(images, gt, label, seed=4)
    assert abs(float(losses[4]) - 3.0 * float(step.ops.rows.mean())) <= 1e-5 * float(losses[4])


def _worker(rank, world, port, out_dir):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        torch.set_num_threads(2)
        images, gt, label = _data(world)
        step = step_of(world, rank, dist)
        losses = step.forward_backward(*(v[rank:rank + 1] for v in (images, gt, label)), seed=4)
        if rank == 0:
            torch.save(dict(grads=_grads(step), losses=losses), os.path.join(out_dir, "dp.pt"))
        dist.barrier()
    finally:
        dist.destroy_process_group()


def test_two_ranks_with_different_numbers_of_rois_give_the_one_rank_gradients(tmp_path):
    mp.spawn(_worker, args=(2, _free_port(), str(tmp_path)), nprocs=2, join=True)
    got = torch.load(tmp_path / "dp.pt", weights_only=True)
    step = step_of(1)
    images, gt, label = _data(2)
    losses, ref = step.forward_backward(images, gt, label, seed=4), _grads(step)
    np.testing.assert_allclose(got["losses"].numpy(), losses.numpy(), rtol=1e-5)
    # float summation order differs (two partial sums added by the all-reduce)
    np.testing.assert_allclose(got["grads"].numpy(), ref.numpy(), rtol=2e-4, atol=1e-6 * float(ref.abs().max()))


@pytest.mark.gpu
def test_the_hip_path_tells_which_rois_are_kept(dev):
    """An NMS threshold so low that images keep few boxes; no gradient of the loss reaches the others' logits."""
    from objectdetection_amd import ops
    from objectdetection_amd.config import PathConfig
    from objectdetection_amd.train import HipPathOps, RPNModel
    torch.manual_seed(0)
    cfg = PathConfig(H=9, W=11, pre_k=500, post_n=150, G=8, nms_thr=0.05)
    rpn = RPNModel(cfg.A, 0.125).to(dev)
    frcn, teacher = (FRCNModel(rpn.channels, 7, n, cfg.num_classes).to(dev) for n in (64, 96))
    with torch.no_grad():
        for m in (*rpn.features, rpn.conv, *frcn.children(), *teacher.children()):
            if hasattr(m, "weight"):
                m.weight.mul_(2.5)             # features and logits of some size, different from RoI to RoI
    path = HipPathOps(cfg, 2, rpn.channels, dev)
    step = TrainStep(rpn, frcn, cfg, path, teacher=teacher)
    images = torch.rand((2, 3, cfg.H * 16 + 8, cfg.W * 16 + 8), device=dev)
    c, half = torch.rand((2, cfg.G, 2), device=dev) * 0.6 + 0.2, torch.rand((2, cfg.G, 2), device=dev) * 0.15 + 0.05
    gt, label = torch.cat([c - half, c + half], -1), torch.randint(0, cfg.num_classes - 1, (2, cfg.G), device=dev)
    losses = step.forward_backward(images, gt, label, seed=1)
    kept = path.path.keep_count.tolist()
    assert all(0 < n < cfg.post_n for n in kept), kept
    with torch.no_grad():
        fmap = rpn(images)[0]
        pooled = path.roi_pool(fmap, path.path.proposed)
        top = tuple(torch.topk(teacher.logits(pooled)[1], 8, -1))
        logits = frcn.logits(pooled)[1]
        rows = ops.distill_loss(logits, *top, temperature=2.0, want_grad=False)["loss"]
    want = float(torch.cat([rows[i, :n] for i, n in enumerate(kept)]).mean())
    # the same kernels on the same inputs; the convolutions may differ in their last bits
    assert abs(float(losses[4]) - want) <= 1e-3 * want and abs(float(rows.mean()) - want) > 0.01 * want
    z = logits.clone().requires_grad_(True)
    w = path.targets(fmap, *rpn(images)[1:], gt, label, 1, 0)["roi_weight"]
    assert [int(v) for v in w.sum(1)] == kept
    g, = torch.autograd.grad(path.distill_loss(z, *top, 2.0, w), z)
    for i, n in enumerate(kept):
        assert not g[i, n:].any() and g[i, :n].any(-1).all()
    assert float(path.distill_loss(z, *top, 2.0, torch.zeros_like(w))) == 0
