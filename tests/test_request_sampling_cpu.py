"""Sampling settings of requests: what they may be, and their way through the scheduler."""
import math

import pytest

from jarvis_b200 import serving


class _Engine:
    def __init__(self):
        self.calls = []

    def admit(self, slot, prompt_tokens, max_new_tokens=0, **own):
        if "sampling" in own:
            serving.check_sampling(own["sampling"])
        self.calls.append((slot, tuple(prompt_tokens), own))

    def release(self, slot):
        pass

    def step(self, active_slots):
        return {s: 7 for s in active_slots}


def test_settings_reach_the_engine_with_the_requests_that_have_them():
    eng = _Engine()
    sched = serving.ContinuousBatchingScheduler(eng, max_batch_size=2)
    mine = {"temperature": 0.5, "min_p": 0.1}
    sched.add_request(serving.Request(0, [1], 2))
    sched.add_request(serving.Request(1, [2], 2, sampling=mine))
    mine["temperature"] = 9.0                                    # the caller's dict is the caller's
    sched.add_request(serving.Request(2, [3], 2, sampling={"top_p": 1.5}))
    sched.run()
    assert eng.calls == [(0, (1,), {}), (1, (2,), {"sampling": {"temperature": 0.5, "min_p": 0.1}})]
    by_id = {r.req_id: r for r in sched.completed}
    assert "top_p" in by_id[2].error and not by_id[2].is_finished and by_id[1].is_finished


def test_settings_that_are_none():
    check = serving.check_sampling
    assert check({}) == {}
    assert check({"temperature": None, "top_k": None, "top_p": None, "min_p": None}) == {"temperature": 0.0, "top_k": 0, "top_p": 0.0, "min_p": 0.0}
    assert check({"temperature": 1, "top_k": 40.0, "top_p": 1}) == {"temperature": 1.0, "top_k": 40, "top_p": 1.0}
    for bad, text in (({"typical_p": 0.5}, "typical_p"), ({"temperature": math.nan}, "finite"), ({"temperature": math.inf}, "finite"), ({"top_k": -1}, "top_k"),
                      ({"top_k": 2.5}, "top_k"), ({"top_k": 2 ** 31}, "top_k"), ({"top_p": -0.1}, "top_p"), ({"top_p": 1.1}, "top_p"), ({"min_p": 2}, "min_p"),
                      ({"top_p": "0.9x"}, "number"), ({"top_k": [1]}, "number")):
        with pytest.raises(ValueError, match=text):
            check(bad)


def test_an_engine_for_all_refuses_a_requests_own_before_it_touches_the_slot():
    eng = serving.CudaDecodeEngine.__new__(serving.CudaDecodeEngine)
    eng.max_position, eng.per_request = 64, False
    with pytest.raises(ValueError, match="per_request"):
        eng.admit(0, [1, 2], max_new_tokens=4, sampling={"temperature": 1.0})
    eng.per_request = True
    with pytest.raises(ValueError, match="min_p"):
        eng.admit(0, [1, 2], max_new_tokens=4, sampling={"min_p": -1.0})


def test_numbers_that_32_bits_do_not_hold_are_refused():
    import torch
    check = serving.check_sampling
    for bad, text in (({"temperature": 1e39}, "finite"), ({"temperature": -1e39}, "finite"), ({"temperature": 10 ** 400}, "number"), ({"top_k": 10 ** 400}, "number"),
                      ({"top_p": torch.zeros(2)}, "number"), ({"min_p": 1j}, "number"), ({1: 2, "x": 3}, "not 1, x")):
        with pytest.raises(ValueError, match=text):
            check(bad)
    assert check({"temperature": torch.finfo(torch.float32).max})["temperature"] == torch.finfo(torch.float32).max


def test_a_request_with_such_settings_does_not_end_the_others():
    sched = serving.ContinuousBatchingScheduler(_Engine(), max_batch_size=2)
    for i, own in enumerate((None, {"temperature": 1e39}, {"top_k": 10 ** 400}, {7: 1.0}, {"top_k": 5})):
        sched.add_request(serving.Request(i, [1], 3, sampling=own))
    sched.run()
    by_id = {r.req_id: r for r in sched.completed}
    assert [by_id[i].error is not None for i in range(5)] == [False, True, True, True, False]
    assert all(by_id[i].is_finished and len(by_id[i].generated_tokens) == 3 for i in (0, 4))


def test_a_released_slot_no_longer_draws_by_the_requests_settings():
    import types

    import torch
    eng = serving.CudaDecodeEngine.__new__(serving.CudaDecodeEngine)
    eng.max_position, eng.per_request, eng.pad_token = 64, True, 0
    eng.defaults = serving.check_sampling(dict(temperature=0.7, top_k=50, top_p=0.9, min_p=None))
    eng.rows = {n: torch.zeros(2, dtype=torch.int32 if n == "top_k" else torch.float32) for n in serving.SAMPLING}
    eng.session = types.SimpleNamespace(state={"h": [torch.zeros(2, 4)], "S": [torch.zeros(2, 1, 2, 2)]}, positions=torch.zeros(2, dtype=torch.int32))
    eng.next_token, eng.active = torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    eng.admit(1, [5], 3, sampling={"top_k": 0, "top_p": 0.95})
    assert eng.rows["temperature"].tolist() == [0.0, pytest.approx(0.7)] and eng.rows["top_k"].tolist() == [0, 0] and eng.active.tolist() == [0, 1]
    eng.release(1)
    assert eng.rows["temperature"].tolist() == [0.0, 0.0] and eng.active.tolist() == [0, 0]
    eng.admit(1, [6], 3)                                          # the engine's own again
    assert eng.rows["temperature"][1] == pytest.approx(0.7) and eng.rows["top_k"][1] == 50 and eng.rows["top_p"][1] == pytest.approx(0.9)
