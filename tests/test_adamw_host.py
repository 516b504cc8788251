"""What ``training.AdamW`` refuses and keeps before any kernel is launched (all on the CPU, where a step ends at the parameters' device)."""
import copy
import io
import threading
import time
import types

import pytest
import torch

from torchtune_amd import AdamW
from torchtune_amd.training import optim


def _saved(p, strides, seed=0):
    """8-bit states of a parameter that lies with these strides"""
    g = torch.Generator().manual_seed(seed)
    code = lambda: torch.randint(0, 128, (p.numel(),), dtype=torch.uint8, generator=g).as_strided(p.shape, strides)
    exponents = torch.randint(90, 120, (-(-p.numel() // 128),), dtype=torch.uint8, generator=g)
    return {"step": 3, "exp_avg": code(), "exp_avg_sq": code(), "exp_avg_exponent": exponents, "exp_avg_sq_exponent": exponents.clone()}


_ROWS, _COLUMNS = (48, 1), (1, 64)


def _parameter(layout):
    return torch.nn.Parameter({"rows": lambda: torch.zeros(64, 48), "columns": lambda: torch.zeros(48, 64).t(),
                               "gaps": lambda: torch.zeros(64, 50)[:, 1:49], "gaps in columns": lambda: torch.zeros(48, 70).t()[3:67],
                               "one row": lambda: torch.zeros(64, 48)[:1], "3d": lambda: torch.zeros(48, 4, 16).permute(1, 2, 0)}[layout]())


@pytest.mark.parametrize("layout,strides,fits", [
    ("rows", _ROWS, True), ("rows", _COLUMNS, False), ("columns", _COLUMNS, True), ("columns", _ROWS, False),
    # a parameter with gaps is copied row by row
    ("gaps", _ROWS, True), ("gaps", _COLUMNS, False), ("gaps in columns", _ROWS, True), ("gaps in columns", _COLUMNS, False),
    ("one row", (48, 1), True), ("one row", (1, 1), True), ("3d", (16, 1, 64), True), ("3d", (768, 48, 1), False),
])
def test_eight_bit_states_of_another_order_in_memory(layout, strides, fits):
    """Their exponents belong to neighbours in memory: refused where those would be others, before anything changes."""
    p = _parameter(layout)
    opt = AdamW([p], state_bits=8)
    saved = {"state": {0: _saved(p, strides)}, "param_groups": opt.state_dict()["param_groups"]}
    with pytest.raises(RuntimeError if fits else ValueError, match="AMD GPU" if fits else "another order"):
        opt.load_state_dict(saved)
    assert fits or not opt.state


def test_flat_eight_bit_states():
    """One after another: right for a parameter whose rows lie that way, and for no other."""
    for layout, fits in (("rows", True), ("gaps", True), ("columns", False)):
        p = _parameter(layout)
        opt = AdamW([p], state_bits=8)
        saved = {"state": {0: {name: t.reshape(-1) if name in ("exp_avg", "exp_avg_sq") else t for name, t in _saved(p, _ROWS).items()}},
                 "param_groups": opt.state_dict()["param_groups"]}
        with pytest.raises(RuntimeError if fits else ValueError, match="AMD GPU" if fits else "another order"):
            opt.load_state_dict(saved)


def test_states_in_32_bits_follow_their_elements():
    """No block, no order: the check lets them through."""
    p = _parameter("rows")
    opt = AdamW([p])
    m = torch.zeros(48, 64).t()
    saved = {"state": {0: {"step": 1, "exp_avg": m, "exp_avg_sq": m}}, "param_groups": opt.state_dict()["param_groups"]}
    with pytest.raises(RuntimeError, match="AMD GPU"):
        opt.load_state_dict(saved)


def test_options_of_a_group_are_checked_and_taken():
    p = lambda: torch.nn.Parameter(torch.zeros(200))
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([{"params": [p()], "state_bits": 16}])
    opt = AdamW([p()])
    with pytest.raises(ValueError, match="state_bits"):
        opt.add_param_group({"params": [p()], "state_bits": 16})
    assert len(opt.param_groups) == 1
    # a group with 8 bits beside one with 32: states of its own width get as far as the device, the other's are refused
    opt = AdamW([{"params": [p()]}, {"params": [p()], "state_bits": 8}])
    eight = _saved(opt.param_groups[1]["params"][0], (1,))
    wide = {"step": 1, "exp_avg": torch.zeros(200), "exp_avg_sq": torch.zeros(200)}
    groups = opt.state_dict()["param_groups"]
    for states, error, match in (({1: eight}, RuntimeError, "AMD GPU"), ({0: wide}, RuntimeError, "AMD GPU"), ({0: eight}, ValueError, "bits"),
                                 ({1: wide}, ValueError, "expected")):
        with pytest.raises(error, match=match):
            opt.load_state_dict({"state": states, "param_groups": groups})


def test_options_of_a_state_dict():
    p = torch.nn.Parameter(torch.zeros(200))
    saved = AdamW([p], lr=0.5, seed=9, stochastic_rounding=True).state_dict()
    opt = AdamW([p], seed=1)
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["seed"] == 9 and opt.param_groups[0]["stochastic_rounding"] and opt.param_groups[0]["lr"] == 0.5
    eight = AdamW([p], state_bits=8)
    eight.load_state_dict(saved)  # no states, nothing to refuse
    assert eight.param_groups[0]["state_bits"] == 8
    # torch's groups know nothing of them
    opt.load_state_dict(torch.optim.AdamW([p], lr=0.25).state_dict())
    assert opt.param_groups[0]["seed"] == 9 and opt.param_groups[0]["stochastic_rounding"] and opt.param_groups[0]["lr"] == 0.25
    assert opt.param_groups[0]["state_bits"] == 32
    with pytest.raises(ValueError):
        opt.load_state_dict({"state": {}, "param_groups": saved["param_groups"] * 2})


def test_a_parameter_replaced_in_its_group():
    """The list is the same and as long, the parameter is another: the native side is made anew."""
    old, new, kept = (torch.nn.Parameter(torch.zeros(4)) for _ in range(3))
    opt = AdamW([old, kept])
    first = opt._plan(0)
    assert opt._plan(0) is first
    opt.param_groups[0]["params"][0] = new
    new.grad = torch.ones(4)
    assert opt._plan(0) is not first
    with pytest.raises(RuntimeError, match="AMD GPU"):  # it is asked for a step
        opt.step()
    opt.param_groups[0]["params"] = [kept]
    opt.step()  # no gradient
    assert opt._plan(0).holds([kept]) and not opt._plan(0).holds([new]) and not opt._plan(0).holds([kept, new]) and not opt._plan(0).holds([None])
    with pytest.warns(UserWarning):
        twice = AdamW([old, old])
    with pytest.raises(ValueError, match="twice"):
        twice.step()


def test_states_taken_out_of_the_dictionary():
    """What the native side holds for them is given up."""
    p = torch.nn.Parameter(torch.zeros(4))
    opt = AdamW([p])
    second = opt._plan(0)
    opt.state = type(opt.state)(dict)  # as empty as the one before
    assert opt._plan(0) is second
    assert not opt.state[torch.nn.Parameter(torch.zeros(1))]  # an entry made by looking for one
    assert len(opt.state) == 1 and opt._plan(0) is second
    opt.state[torch.nn.Parameter(torch.zeros(1))] = {"step": 1}
    assert opt._plan(0) is not second


@pytest.mark.parametrize("what", ["parameter", "gradient"])
@pytest.mark.parametrize("elements", [0, 99])
def test_memory_that_has_been_given_up(what, elements):
    """A storage resized under a tensor: refused, before the device is looked at; one that is whole gets that far."""
    p = torch.nn.Parameter(torch.zeros(120)[20:].view(10, 10))
    p.grad = torch.ones(10, 11)[:, 1:]
    opt = AdamW([p])
    t = p if what == "parameter" else p.grad
    whole = t.untyped_storage().nbytes()
    with pytest.raises(RuntimeError, match="AMD GPU"):
        opt.step()
    t.untyped_storage().resize_(elements * 4)
    with pytest.raises(RuntimeError, match=f"memory of a {what}"):
        opt.step()
    t.untyped_storage().resize_(whole)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        opt.step()


def _views(base, *places):
    return [torch.nn.Parameter(base.as_strided(size, stride, offset)) for size, stride, offset in places]


@pytest.mark.parametrize("places,shared", [
    # one after another, an empty one among them; the same twice; by one element; a part of a larger one
    ([((10,), (1,), 0), ((0,), (1,), 5), ((10,), (1,), 10), ((4, 5), (5, 1), 20)], None),
    ([((10,), (1,), 30), ((10,), (1,), 0), ((10,), (1,), 30)], (0, 2)),
    ([((10,), (1,), 9), ((10,), (1,), 0)], (0, 1)),
    ([((100,), (1,), 0), ((4, 5), (5, 1), 20), ((1,), (1,), 200)], (0, 1)),
    # columns of one matrix of pitch 20, that begin anywhere; by one column; the last columns with the first of the next row
    ([((10, 5), (20, 1), 7), ((10, 8), (20, 1), 12), ((10, 7), (20, 1), 0)], None),
    ([((10, 5), (20, 1), 7), ((10, 8), (20, 1), 11)], (0, 1)),
    ([((10, 5), (20, 1), 18), ((10, 8), (20, 1), 3)], None),
    ([((10, 6), (20, 1), 18), ((10, 8), (20, 1), 3)], (0, 1)),
    # transposed columns, single columns, interleaved elements, columns of one matrix in three dimensions
    ([((5, 10), (1, 20), 0), ((8, 10), (1, 20), 5)], None),
    ([((10,), (20,), 3), ((10,), (20,), 4), ((10, 3), (20, 1), 5)], None),
    ([((50,), (2,), 0), ((50,), (2,), 1)], None),
    ([((50,), (2,), 0), ((50,), (2,), 2)], (0, 1)),
    ([((4, 5, 3), (100, 20, 1), 0), ((4, 5, 17), (100, 20, 1), 3)], None),
    ([((4, 2, 20), (100, 20, 1), 0), ((4, 3, 20), (100, 20, 1), 40)], None),
    # rows in between, in the same columns: the same places modulo the pitch of a row, others modulo that of two
    ([((5, 8), (40, 1), 0), ((5, 8), (40, 1), 20)], None),
    # elements of the one are in the gaps of the other, but along no dimension: not seen
    ([((5,), (4,), 0), ((5,), (6,), 1)], (0, 1)),
])
def test_parameters_that_share_memory(places, shared):
    from torchtune_amd import _host

    params = _views(torch.zeros(400), *places)
    assert _host.load().overlapping(params) == shared
    assert _host.load().overlapping(params[::-1]) == (None if shared is None else tuple(sorted(len(params) - 1 - i for i in shared)))
    # by the elements themselves
    marks = [torch.zeros(400, dtype=torch.bool) for _ in places]
    for m, (size, stride, offset) in zip(marks, places):
        m.as_strided(size, stride, offset).fill_(True)
    if shared is None:
        assert int(sum(m.int() for m in marks).max()) <= 1
    elif places[0][1] != (4,):
        assert bool((marks[shared[0]] & marks[shared[1]]).any())


@pytest.mark.parametrize("call", ["step", "moments", "state_dict"])
def test_threads_make_one_native_side(call, monkeypatch):
    """The first calls of several threads, while making it takes its time."""
    real, made = optim._host.load(), []

    def slowly(*args):
        made.append(threading.get_ident())
        time.sleep(0.05)
        return real.AdamWGroup(*args)

    monkeypatch.setattr(optim._host, "load", lambda: types.SimpleNamespace(AdamWGroup=slowly, adamw_step=real.adamw_step))
    opt = AdamW([torch.nn.Parameter(torch.zeros(4))])
    start = threading.Barrier(4)

    def work(i):
        start.wait()
        if call == "step" or i % 2:
            opt.step()
        elif call == "state_dict":
            opt.state_dict()
        else:
            with pytest.raises(RuntimeError, match="no parameter"):
                opt.moments()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1


def test_a_copy_has_a_lock_of_its_own():
    opt = AdamW([torch.nn.Parameter(torch.zeros(4))])
    f = io.BytesIO()
    torch.save(opt, f)
    f.seek(0)
    for other in (copy.deepcopy(opt), torch.load(f, weights_only=False)):  # written three lines above
        other.step()
        assert other._lock is not opt._lock
    lock = opt._lock
    opt.load_state_dict(opt.state_dict())
    assert opt._lock is lock


def test_hooks_of_a_load():
    """Hooks before it see the states and may change them; what is checked is what they leave."""
    p = torch.nn.Parameter(torch.zeros(200))
    saved = {"state": {0: {"step": 1, "exp_avg": torch.zeros(200), "exp_avg_sq": torch.zeros(200)}}, "param_groups": AdamW([p]).state_dict()["param_groups"]}
    opt, seen = AdamW([p]), []

    def look(o, d):
        seen.append(sorted(d["state"]))

    def drop(o, d):
        return {**d, "state": {}}

    def spoil(o, d):
        return {**d, "state": {0: {"step": 1}}}

    opt.register_load_state_dict_pre_hook(look)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        opt.load_state_dict(saved)
    handle = opt.register_load_state_dict_pre_hook(spoil)
    with pytest.raises(ValueError, match="expected"):
        opt.load_state_dict(saved)
    handle.remove()
    opt.register_load_state_dict_pre_hook(drop)
    opt.register_load_state_dict_pre_hook(look)
    opt.register_load_state_dict_post_hook(lambda o: seen.append("after"))
    opt.load_state_dict(saved)
    assert seen == [[0], [0], [0], [], "after"] and sorted(saved["state"]) == [0]
    opt.load_state_dict(saved)
    assert len(seen) == 8 and not opt.state


def test_a_width_written_into_a_group():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = AdamW([p])
    opt.param_groups[0]["state_bits"] = 16
    with pytest.raises(ValueError, match="state_bits"):
        opt.step()
    opt.param_groups[0]["state_bits"] = 8  # no states yet
    opt.step()
    with pytest.raises(TypeError):
        opt.add_param_group([p])
