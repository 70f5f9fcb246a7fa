"""Host logic around the capture of a step, on the CPU."""


def test_a_capture_waits_for_the_watchdog_only_where_there_is_one(monkeypatch):
    """GraphedStep empties the RCCL group's list of collectives before it captures: the watchdog's queries of theirs would abort the process"""
    import torch.distributed as dist

    from uemda_amd.step import retire_collectives
    assert not dist.is_initialized() and retire_collectives() is False
    calls = []

    class World:
        def _wait_for_pending_works(self):
            calls.append(1)
    assert hasattr(dist.ProcessGroup, "_wait_for_pending_works")
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_backend", lambda: "gloo")
    assert retire_collectives() is False and not calls
    monkeypatch.setattr(dist, "get_backend", lambda: "nccl")
    monkeypatch.setattr(dist, "group", type("group", (), {"WORLD": World()}))
    assert retire_collectives() is True and calls == [1]
