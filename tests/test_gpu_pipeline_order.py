"""What the caller has queued to read of a call is not overwritten: with one batch at a time and inputs that
are ready before the call by the training targets, which have a stream of their own, and by calls made
on another stream."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def batches(dev, n, seed=40):
    from oracle import frcnn_oracle as O
    from objectdetection_amd.config import PathConfig
    cfg = PathConfig(H=16, W=20, pre_k=1000, post_n=200, G=8)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)
    data = []
    for i in range(n):
        d = O.synth_inputs(seed=seed + i, B=2, H=cfg.H, W=cfg.W, A=cfg.A, C=32, G=cfg.G)
        data.append([t(d[k]) for k in ("fmap", "score", "coord", "gt", "label")])
    return cfg, data


def results(path):
    return [t.clone() for t in (path.rpn["pos"], path.rpn["reg"], path.proposed, path.tindex, path.gt_coord, path.pooled)]


def expected(cfg, data, dev):
    from objectdetection_amd.pipeline import RegionProposalPath
    plain, ref = RegionProposalPath(cfg, 2, 32, dev, train=True, depth=1), []
    for i, x in enumerate(data):
        plain.run(*x, seed=i)
        torch.cuda.synchronize()
        ref.append(results(plain))
    return ref


def test_late_reads_with_one_batch_at_a_time(dev):
    from objectdetection_amd.pipeline import RegionProposalPath
    cfg, data = batches(dev, 4)
    ref = expected(cfg, data, dev)
    for _ in range(3):                       # other streams each time: some share a hardware queue
        path, got = RegionProposalPath(cfg, 2, 32, dev, train=True, depth=1), []
        torch.cuda.synchronize()
        ready = torch.cuda.Event()
        ready.record()
        for i, x in enumerate(data):
            path.run(*x, seed=i, inputs_ready=ready)
            torch.cuda._sleep(3_000_000)     # the reads come late, the host is far ahead
            got.append(results(path))
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, ref)):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), i


@pytest.mark.parametrize("depth", [1, 2])
def test_calls_on_two_streams_in_turn(dev, depth):
    """The caller orders nothing between them, also through the function that keeps its buffers by itself."""
    from objectdetection_amd import pipeline
    from objectdetection_amd.module import process_fmap
    cfg, data = batches(dev, 6)
    ref = expected(cfg, data, dev)
    path, got = pipeline.RegionProposalPath(cfg, 2, 32, dev, train=True, depth=depth), []
    pipeline.clear_path_cache()
    torch.cuda.synchronize()
    ready = torch.cuda.Event()
    ready.record()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, x in enumerate(data):
        with torch.cuda.stream(streams[i % 2]):
            path.run(*x, seed=i, inputs_ready=ready)
            torch.cuda._sleep(2_000_000)
            got.append(results(path))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(got, ref)):
        assert all(torch.equal(x, y) for x, y in zip(a, b)), i
    got = []
    for i, (fmap, score, coord, _, _) in enumerate(data):
        with torch.cuda.stream(streams[i % 2]):
            crop, proposed = process_fmap(fmap, score, coord, path.anchor.view(cfg.H, cfg.W, cfg.A, 4), cfg, fuse_pool=True,
                                          inputs_ready=ready)
            torch.cuda._sleep(2_000_000)
            got.append((crop.clone(), proposed.clone()))
    torch.cuda.synchronize()
    for i, ((crop, proposed), b) in enumerate(zip(got, ref)):
        assert torch.equal(proposed, b[2]) and torch.equal(crop, b[5]), i
    pipeline.clear_path_cache()


def test_captures_between_calls_on_other_streams(dev):
    """A path that has run on two streams is captured, replayed and run again."""
    from objectdetection_amd.pipeline import RegionProposalPath
    cfg, data = batches(dev, 3)
    ref = expected(cfg, data, dev)
    path = RegionProposalPath(cfg, 2, 32, dev, train=True, depth=1)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            path.run(*data[i], seed=i)
            torch.cuda._sleep(1_000_000)
    graph = path.capture(*data[2], seed=2)
    for i in (0, 1, 0):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(results(path), ref[2]))
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[i]):
            path.run(*data[i], seed=i)
            got = results(path)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ref[i])), i
