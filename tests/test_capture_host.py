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


def test_a_capture_waits_for_every_group_of_rccl(monkeypatch):
    """an Aligner's or a ClassBalance's own process group has a watchdog of its own, beside the world's, whatever the world's backend is"""
    import torch.distributed as dist

    from uemda_amd.step import retire_collectives
    calls = []

    class Group:
        def __init__(self, name):
            self.name = name

        def _wait_for_pending_works(self):
            calls.append(self.name)
    world, one, two, host = (Group(n) for n in ("world", "one", "two", "host"))
    groups = {world: ("nccl", None), one: ("nccl", None), host: ("gloo", None), two: ("nccl", None)}
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_backend", lambda group=None: groups[group or world][0])
    monkeypatch.setattr(dist, "group", type("group", (), {"WORLD": world}))
    monkeypatch.setattr(dist.distributed_c10d, "_world", type("world", (), {"pg_map": groups}))
    assert retire_collectives() is True and sorted(calls) == ["one", "two", "world"]
    groups[world] = ("gloo", None)
    calls.clear()
    assert retire_collectives() is True and sorted(calls) == ["one", "two"]
    del groups[one], groups[two]
    calls.clear()
    assert retire_collectives() is False and not calls


def test_groups_of_a_real_backend_are_seen(tmp_path):
    """the table of groups that the wait goes through holds the world's group and one made beside it, by backend"""
    import subprocess
    import sys
    code = f"""if True:
        import torch.distributed as dist
        from uemda_amd.step import retire_collectives
        dist.init_process_group("gloo", init_method="file://{tmp_path}/store", rank=0, world_size=1)
        side = dist.new_group([0])
        table = dict((g, b) for g, (b, _) in dist.distributed_c10d._world.pg_map.items())
        assert table[dist.group.WORLD] == table[side] == "gloo" and len(table) == 2, table
        assert retire_collectives() is False
        dist.destroy_process_group()
    """
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stderr[-2000:]
