"""Rotary positions: arrays that are written and read by the same call."""
import pytest
import torch

from sddmm_gpu_b200 import api

pytestmark = pytest.mark.gpu


def _x(*shape):
    return torch.randn(shape, device="cuda")


def test_arrays_that_race_are_refused(engine):
    f = api.rotary_frequencies(64)
    x, y, z = _x(10, 2, 64), _x(10, 2, 64), _x(20, 2, 64)
    rows = torch.arange(10, device="cuda")
    part = api.RotaryPart
    wide = torch.as_strided(x, (4, 2, 64), (128, 64, 1))
    for parts in ([part(x, y), part(y, z[:10])],                      # reads what the other writes
                  [part(y, z[:10]), part(x, y)],
                  [part(x), part(x, y)],                              # in place, and read by another
                  [part(x, z[:10]), part(y, z[:10])],                 # both write z
                  [part(x, z[:10]), part(y, z, rows)],
                  [part(x, z, rows), part(y, z, rows)],               # the same rows of z
                  [part(z[:10], z, rows)],                            # listed rows of what it reads
                  [part(wide, torch.as_strided(x, (4, 2, 64), (64, 256, 1)))],   # other strides over the same memory
                  [part(x, y), part(x, y, rotate=False)]):
        before = [t.clone() for t in (x, y, z)]
        with pytest.raises(api.SddmmError) as e:
            engine.rotary(parts, 0, f)
        assert e.value.status == api.INVALID_ARG
        assert all(torch.equal(a, b) for a, b in zip(before, (x, y, z)))


def test_arrays_that_do_not_race_are_taken(engine):
    f = api.rotary_frequencies(64)
    x, y = _x(10, 2, 64), _x(10, 2, 64)
    part = api.RotaryPart
    want = [torch.empty_like(x) for _ in range(2)]
    engine.rotary([part(x, want[0]), part(y, want[1])], 3, f)
    # one source twice; two lists of one cache; halves of one buffer, in place; nothing written where nothing is to be done
    a, b = torch.empty_like(x), torch.empty_like(x)
    engine.rotary([part(x, a), part(x, b, rotate=False)], 3, f)
    assert torch.equal(a, want[0]) and torch.equal(b, x)
    cache = torch.zeros((40, 2, 64), device="cuda")
    engine.rotary([part(x, cache, torch.arange(10, device="cuda")), part(y, cache, torch.arange(10, device="cuda") + 20)], 3, f)
    assert torch.equal(cache[:10], want[0]) and torch.equal(cache[20:30], want[1]) and not bool(cache[10:20].any())
    both = torch.cat([x, y], 1)
    engine.rotary([part(both[:, :2]), part(both[:, 2:])], 3, f)
    assert torch.equal(both, torch.cat(want, 1))
    engine.rotary([part(x, rotate=False), part(x, a)], 3, f)
    assert torch.equal(a, want[0])
