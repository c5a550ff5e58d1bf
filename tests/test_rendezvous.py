"""The port that the benchmark's ranks agree on: through the store, without a process group -- the run's own group is the first and only one that
leaves addresses there."""
import importlib.util
import os
import socket
import subprocess
import sys
import threading

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load_bench():
    spec = importlib.util.spec_from_file_location("bench_under_test", os.path.join(ROOT, "bench.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def test_the_port_is_agreed_without_a_process_group(monkeypatch):
    import torch.distributed as dist

    def refuse(*args, **kwargs):
        raise AssertionError("a process group for the port")

    ports = iter(range(20001, 20100))        # (which of the calls a port is from has to show)
    monkeypatch.setattr(dist, "init_process_group", refuse)
    monkeypatch.setenv("MASTER_ADDR", "127.0.0.1")
    monkeypatch.setenv("MASTER_PORT", str(free_port()))
    monkeypatch.delenv("TORCHELASTIC_USE_AGENT_STORE", raising=False)
    ranks = [load_bench(), load_bench()]     # (a module of its own for each: they keep their stores)
    got = [None, None]
    monkeypatch.setattr(ranks[0], "_free_port", lambda: next(ports))

    def run(rank):
        try:
            got[rank] = [ranks[rank].agree_on_port(2, rank) for _ in range(3)]
        except BaseException as e:    # (raised in a thread: shown by the comparison below)
            got[rank] = e

    threads = [threading.Thread(target=run, args=(r,), daemon=True) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert got[0] == got[1] == [20001, 20002, 20003], got
    assert load_bench().agree_on_port(1, 0) > 0


def test_ranks_without_an_agent_store(tmp_path):
    """the ranks started by hand (no launcher that serves the store: rank 0 does): they agree, meet and end"""
    env = {k: v for k, v in os.environ.items() if not k.startswith("TORCHELASTIC_")}
    env.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(free_port()), WORLD_SIZE="2", EMX_BENCH_WATCHDOG="60")
    procs = [subprocess.Popen([sys.executable, os.path.join(ROOT, "bench.py"), "--gpus", "2", "--launch-check"], cwd=str(tmp_path),
                              env=dict(env, RANK=str(r), LOCAL_RANK=str(r)), stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True) for r in range(2)]
    out = []
    try:
        for p in procs:
            out.append(p.communicate(timeout=120))
    finally:
        for p in procs:
            p.kill()
    assert [p.returncode for p in procs] == [0, 0], [o[1][-1000:] for o in out]
    assert '"probe_port_agreed": true' in out[0][0]
