"""What adapters and beams refuse, checked where no GPU is needed."""

from __future__ import annotations

import pytest
import torch

from kvforge_b200 import ops

BF = torch.bfloat16


def bank_args(s=2, sections=2, r=16, k=64, n=64, dtype=BF):
    return [torch.zeros(s, sections, r, k, dtype=dtype), torch.zeros(s, n, r, dtype=dtype), torch.ones(s)]


def test_adapter_bank_refusals():
    ops.AdapterBank(*bank_args(), ends=(24, 64))
    a, b, sc = bank_args()
    for bad in (
        dict(a=a.half(), b=b.half()), dict(a=a.float()), dict(a=a[0]), dict(b=b[:, :, :8]), dict(b=b[:1]), dict(a=a.transpose(2, 3)), dict(scales=sc.double()),
        dict(scales=sc[:1]), dict(ends=(64,)), dict(ends=(64, 24)), dict(ends=(0, 64)), dict(ends=(20, 64)), dict(ends=(24, 56)), dict(ends=(64, 64)),
        dict(alternating=True), dict(ranks=torch.ones(2)), dict(ranks=torch.ones(1, dtype=torch.int32)),
    ):  # fmt: skip
        args = {"a": a, "b": b, "scales": sc, "ends": (24, 64), **bad}
        with pytest.raises((ValueError, TypeError)):
            ops.AdapterBank(**args)
    for kw in (dict(r=8), dict(r=144), dict(sections=4, r=112), dict(sections=5), dict(k=60), dict(n=60), dict(s=0)):
        c = bank_args(**kw)
        with pytest.raises((ValueError, TypeError)):
            ops.AdapterBank(*c, ends=tuple(range(8, 8 * c[0].shape[1], 8)) + (c[1].shape[1],))


def test_adapter_call_refusals():
    bank = ops.AdapterBank(*bank_args(sections=1))
    groups = ops.AdapterGroups(8, 2, "cpu")
    ids = torch.zeros(4, dtype=torch.int32)
    for bad in (ids.long(), ids[None], torch.zeros(9, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            ops.group_by_adapter(bad, groups)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.group_by_adapter(ids, groups)
    x, out = torch.zeros(4, 64, dtype=BF), torch.zeros(4, 64, dtype=BF)
    with pytest.raises(ValueError, match="groups"):
        ops.adapter_add(x, bank, groups, out)
    groups.ids, groups.n = ids, 4
    for x_, out_, base_ in (
        (x.float(), out, None), (x[:3], out, None), (x[:, :56], out, None), (x, out[:3], None), (x, out.half(), None), (x, out, out.float()), (x, out, out[:, :56]),
        (torch.zeros(4, 72, dtype=BF)[:, 4:68], out, None), (torch.zeros(4, 68, dtype=BF)[:, :64], out, None), (torch.zeros(64, 4, dtype=BF).t(), out, None),
        (x, torch.zeros(4, 68, dtype=BF)[:, :64], None), (x, torch.zeros(64, 4, dtype=BF).t(), None),
    ):  # fmt: skip
        with pytest.raises(ValueError):
            ops.adapter_add(x_, bank, groups, out_, base=base_)
    for x_, out_, base_ in ((x[:1].expand(4, 64), out, None), (x, out[:1].expand(4, 64), None), (x, out, out[:1].expand(4, 64))):  # rows that are one
        with pytest.raises(ValueError):
            ops.adapter_add(x_, bank, groups, out_, base=base_)
    with pytest.raises(ValueError, match="groups"):
        ops.adapter_add(x, ops.AdapterBank(*bank_args(s=3, sections=1)), groups, out)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.adapter_add(x, bank, groups, out)
    with pytest.raises(ValueError):
        ops.AdapterGroups(0, 1, "cpu")


def test_beam_select_refusals():
    def args(rows=8, v=50, prompts=2, k=6):
        i = lambda: torch.zeros(prompts, k, dtype=torch.int32)  # noqa: E731
        return dict(logits=torch.zeros(rows, v), scores=torch.zeros(rows), parents=i(), tokens=i(), best=torch.zeros(prompts, k), workspace=ops.beam_workspace(rows, v, k, "cpu"))

    with pytest.raises(RuntimeError, match="CUDA"):
        ops.beam_select(**args())
    good = args()
    for bad in (
        dict(logits=good["logits"].double()), dict(logits=good["logits"][0]), dict(logits=torch.zeros(50, 8).t()), dict(logits=torch.zeros(7, 50)), dict(scores=torch.zeros(7)),
        dict(scores=torch.zeros(8).double()), dict(tokens=torch.zeros(2, 5, dtype=torch.int32)), dict(parents=torch.zeros(2, 6)), dict(best=torch.zeros(2, 6).double()),
        dict(workspace=torch.zeros(3, dtype=torch.int64)), dict(workspace=torch.zeros(4096)), dict(logits=torch.zeros(8, 1).expand(8, 50)), dict(parents=torch.zeros(0, 6, dtype=torch.int32)),
    ):  # fmt: skip
        with pytest.raises((ValueError, TypeError)):
            ops.beam_select(**{**good, **bad})
    for kw in (dict(rows=130), dict(k=65), dict(k=0)):
        with pytest.raises(ValueError):
            ops.beam_select(**args(**kw))


def test_copy_refusals():
    k = torch.zeros(2, 4, 2, 8, 16)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.copy_pages(k, k.clone(), i, i)
    for bad in (
        dict(k=k[0]), dict(v=k[:, :3]), dict(v=k.bfloat16()), dict(k=k.transpose(3, 4)), dict(src=i.long()), dict(dst=i[:2]), dict(tokens=i[:2]), dict(tokens=i.long()),
        dict(src=torch.zeros(6, dtype=torch.int32)[::2]),
    ):  # fmt: skip
        with pytest.raises(ValueError):
            ops.copy_pages(**{**dict(k=k, v=None, src=i, dst=i, tokens=None), **bad})
    s = torch.zeros(4, 10)
    for bad in ([], [s, torch.zeros(5, 10)], [s.t()], [torch.zeros(4, 0)], [torch.zeros(1, 10).expand(4, 10)]):
        with pytest.raises(ValueError):
            ops.StateTable(bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.StateTable([s])
