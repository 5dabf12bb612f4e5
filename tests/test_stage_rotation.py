"""The staging buffers of the peer-memory reduce-scatter, in whatever order units come: a buffer may be written again after two other units at the earliest,
since a member has folded a unit when it publishes the next one, and that is only waited for before the one after it."""

from types import SimpleNamespace

import pytest
import torch

from olmax_b200.parallel.symm import SymmContext


class _Barrier:
    def __init__(self):
        self.epoch = 0

    def arrive(self):
        self.epoch += 1
        return self.epoch

    def wait(self, token):
        pass


def _context(monkeypatch, folds):
    ctx = SymmContext.__new__(SymmContext)
    ctx.R, ctx.rank, ctx.stage_slot, ctx.wire_bytes = 2, 1, 16, 2
    ctx.stage_ptrs, ctx._tables, ctx._rs_pending, ctx._barrier = [0, 10 ** 6], {}, None, _Barrier()
    ctx._stage_next, ctx._stage_of = -1, {}
    ctx.rs_stage = torch.arange(ctx.N_STAGE * ctx.R * ctx.stage_slot)
    ctx.grad = torch.zeros(64)
    ctx.store = SimpleNamespace(device=torch.device("cpu"), grad_scale=1.0)
    monkeypatch.setattr("olmax_b200.parallel.symm.K.reduce_slots",
                        lambda stage, acc, n, R, slot, scale: folds.append(int(stage[0]) // (ctx.R * ctx.stage_slot)))
    return ctx


def _unit(index):
    unit = SimpleNamespace(index=index, _staged=set(), params=[])
    for i in range(2):
        unit.params.append(SimpleNamespace(name=f"{index}.{i}", unit=unit, meta=SimpleNamespace(unit_offset=8 * i, offset=0, numel_local=8)))
    return unit


def _stage(ctx, unit):
    """Both weights of a unit; the buffer that both went to on both members."""
    found = set()
    for h in unit.params:
        table = ctx.stage_pointer_table(h).tolist()
        for base, at in zip(ctx.stage_ptrs, table):
            slot, offset = divmod((at - base) // ctx.wire_bytes, ctx.stage_slot)
            assert offset == h.meta.unit_offset and slot % ctx.R == ctx.rank
            found.add(slot // ctx.R)
        unit._staged.add(h.name)
    assert len(found) == 1
    return found.pop()


@pytest.mark.parametrize("layers", [1, 2, 3, 4, 5, 6])
def test_three_stagings_in_a_row_use_three_buffers(monkeypatch, layers):
    folds, stagings = [], []
    ctx = _context(monkeypatch, folds)
    units = [_unit(i) for i in range(layers + 2)]          # the embedding, which stages nothing, the layers, the head
    head, backward = units[-1], units[-2:0:-1]

    def done(unit, flush=False):
        names, unit._staged = unit._staged, set()
        ctx.rs_unit_done(unit, names)
        if flush:
            ctx.rs_flush()

    for two_passes in (False, False, True):
        for _ in range(2 if two_passes else 1):             # two forward passes, one backward pass of both
            stagings.append(_stage(ctx, head))              # folded at once
            done(head, flush=True)
            for unit in backward:
                stagings.append(_stage(ctx, unit))
                done(unit)
        ctx.rs_flush()                                      # the end of the backward pass
    assert folds[::2] == folds[1::2] == stagings            # every unit is folded from where it was staged, in order
    for i in range(2, len(stagings)):
        assert len(set(stagings[i - 2 : i + 1])) == 3, stagings
