"""Whether two uses of a buffer of RegionProposalPath, one of them a write, are ordered: the path's calls
on streams and events that only keep account (no GPU).  An event holds what its stream had done when it was
recorded; a stream that waits for it has that behind it."""
import pytest
import torch

from objectdetection_amd import pipeline
from objectdetection_amd.config import PathConfig

WRITES = {          # the arguments each entry point writes, by the names of the path's buffers
    "frcnn_topk_sort": {"top_scores", "top_idx", "cand", "topk_ws"},
    "frcnn_nms": {"proposed", "keep_pos", "keep_count", "nms_ws"},
    "frcnn_nms_fused": {"proposed", "keep_pos", "keep_count", "nms_ws"},
    "frcnn_iou_assign": {"max_iou", "best_gt", "flags"},
    "frcnn_rpn_sample": {"rpn.label", "rpn.anchor", "rpn.gt", "rpn.gt_list", "rpn.pos", "rpn.reg", "rpn.counts"},
    "frcnn_roi_fwd_prepare": {"roi_ws"},
    "frcnn_label_proposals": {"p_label", "gt_mask", "gt_onehot", "gt_coord", "p_best", "p_iou"},
    "frcnn_sample_proposals": {"tindex", "head_counts"},
    "frcnn_roi_crop_pool_fwd_prepared": {"pooled", "winner"},
}
RESULTS = ("proposed", "keep_count", "tindex", "gt_onehot", "gt_coord", "gt_mask", "pooled", "rpn.pos", "rpn.reg")


class Account:
    """What has happened: uses of buffers, each with all that was behind it."""

    def __init__(self):
        self.streams, self.uses, self.current, self.number = [], [], None, 0

    def use(self, stream, what, buffers):
        """buffers: {address: written}"""
        me = self.number
        self.number += 1
        for address, written in buffers.items():
            for other, name, wrote, n in [u for u in self.uses if u[0] == address]:
                if (written or wrote) and n not in stream.behind:
                    raise AssertionError(f"{what} and {name} use the same buffer without an order")
            self.uses.append((address, what, written, me))
        stream.behind.add(me)


ACC = None


class Stream:
    def __init__(self, device=None):
        self.behind = set()
        ACC.streams.append(self)
        self.cuda_stream = 1000 + len(ACC.streams)

    def wait_event(self, e):
        self.behind |= e.held

    def wait_stream(self, s):
        self.behind |= s.behind


class Event:
    def __init__(self):
        self.held = set()

    def record(self, stream):
        self.held = set(stream.behind)


class Library:
    """Entry points that take part in the account instead of launching anything."""

    def __init__(self, names):
        self.names = names                     # address -> name, filled by the test

    def __getattr__(self, fn):
        def call(*args):
            stream = next(s for s in ACC.streams if s.cuda_stream == args[-1])
            held = {}
            for a in args[:-1]:
                address = getattr(a, "value", None)
                if address in self.names:
                    held[address] = self.names[address] in WRITES[fn]
            ACC.use(stream, fn, held)
            return 1 if fn == "frcnn_roi_fwd_prepare" else 0
        return call


@pytest.fixture
def account(monkeypatch):
    global ACC
    ACC = Account()
    ACC.current = Stream()
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: ACC.current)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(pipeline.ops, "anchors", lambda *a: torch.zeros((16 * 20 * 9, 4)))
    names = {}
    monkeypatch.setattr(pipeline, "lib", Library(names))
    yield ACC, names


def build(names, **how):
    cfg = PathConfig(H=16, W=20, pre_k=200, post_n=40, G=8)
    path = pipeline.RegionProposalPath(cfg, 2, 8, "cpu", **how)
    for d in path._sets:
        for k, v in d.items():
            if k == "rpn":
                names.update({t.data_ptr(): "rpn." + n for n, t in v.items()})
            elif k != "ev":
                names[v.data_ptr()] = k
    for k in ("pooled", "winner"):
        if getattr(path, k) is not None:
            names[getattr(path, k).data_ptr()] = k
    z = lambda *s: torch.zeros(s)
    ins = [z(2, 16, 20, 8), z(2, 16, 20, 9), z(2, 16, 20, 36)]
    return path, ins + ([z(2, 8, 4), torch.zeros((2, 8), dtype=torch.int64)] if how.get("train") else [])


def read(path, names, stream):
    """The caller queues reads of the call's results on `stream`."""
    held = {}
    for name in RESULTS:
        t = path
        for part in name.split("."):
            t = t[part] if isinstance(t, dict) else getattr(t, part, None)
            if t is None:
                break
        else:
            held[t.data_ptr()] = False
    ACC.use(stream, "the caller's read", held)


@pytest.mark.parametrize("depth", [1, 2])
@pytest.mark.parametrize("train,rpn", [(True, True), (True, False), (False, False)])
@pytest.mark.parametrize("given", [True, False])
@pytest.mark.parametrize("streams", [1, 2, 3])
def test_every_two_uses_are_ordered(account, depth, train, rpn, given, streams):
    """Calls on one stream or on several in turn (which the caller does not order), with inputs that are ready
    from the start or where the caller's stream stands; the results are read before the next call, on the stream of the call."""
    acc, names = account
    path, ins = build(names, depth=depth, train=train, rpn_targets=rpn)
    ready = Event()
    callers = [acc.current] + [Stream() for _ in range(streams - 1)]
    for n in range(9):
        acc.current = callers[n % streams]
        path.run(*ins, seed=n, inputs_ready=ready if given else None)
        read(path, names, acc.current)


@pytest.mark.parametrize("depth", [1, 2])
def test_reads_on_the_next_calls_stream(account, depth):
    """The results are read by the stream that makes the next call, which waits for the one before."""
    acc, names = account
    path, ins = build(names, depth=depth, train=True)
    ready, callers = Event(), [acc.current, Stream()]
    for n in range(7):
        acc.current = callers[n % 2]
        path.run(*ins, inputs_ready=ready)
        callers[(n + 1) % 2].wait_stream(callers[n % 2])
        read(path, names, callers[(n + 1) % 2])


def test_the_account_sees_an_order_that_is_missing(account):
    """A planted mistake: a reader on a stream that waits for nothing."""
    acc, names = account
    path, ins = build(names, depth=2, train=True)
    path.run(*ins)
    with pytest.raises(AssertionError, match="without an order"):
        read(path, names, Stream())
