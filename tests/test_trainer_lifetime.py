"""When and where a trainer and the graphs that it captured end: at once, where the last reference goes, and never inside a capture.
A captured graph's end waits for the device and gives its memory pool back; left to the cyclic collector it comes on whichever thread
allocates next (the batch feeder's, autograd's) and while another graph is being captured."""
import contextlib
import gc
import os
import subprocess
import sys
import threading
import types

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# A trainer on the CPU device model (tests/emu/harness.py): replayed steps, then its last reference goes with the collector off.
LIFETIME = '''
import gc, os, sys, weakref
sys.path[:0] = [{root!r}, os.path.join({root!r}, 'tests'), os.path.join({root!r}, 'tests', 'emu')]
import harness
harness.install()
import torch
import test_gpu_step as T
from oracle import s2ag_oracle as O
from s2ag_testing import to_cuda
gc.collect()
gc.disable()
for step in ('eager', 'graph'):
    pr, _ = T.make_processor(32, 64, 12, 2, 9000, 0.3, hip_graph=step == 'graph')
    b = to_cuda(O.recipe_inputs(2, 34, 9100, 64, 12))
    pr.train_step(b['in_text'], b['in_audio'], b['in_mfcc'], b['target'], b['vid'])
    held = [weakref.ref(pr)] + ([weakref.ref(pr._graphed['segs'])] if step == 'graph' else [])
    del pr
    print(step, 'LEFT', sum(r() is not None for r in held), flush=True)
'''


def test_a_trainer_and_its_graphs_end_without_the_collector():
    env = dict(os.environ, S2AG_EMU='1')
    env.pop('S2AG_HIP_LIB', None)
    p = subprocess.run([sys.executable, '-c', LIFETIME.format(root=ROOT)], env=env, capture_output=True, text=True, timeout=900, cwd=ROOT)
    assert p.returncode == 0, p.stderr[-3000:]
    assert [ln for ln in p.stdout.splitlines() if 'LEFT' in ln] == ['eager LEFT 0', 'graph LEFT 0']


class _Stream:
    def wait_stream(self, s):
        pass


@pytest.fixture
def fake_runtime(monkeypatch):
    """torch.cuda's capture as inert objects; ``inside`` is true between the begin and the end of one."""
    state = types.SimpleNamespace(inside=False)

    @contextlib.contextmanager
    def graph(g, pool=None, capture_error_mode='global'):
        assert capture_error_mode == 'thread_local'
        state.inside = True
        try:
            yield
        finally:
            state.inside = False
    monkeypatch.setattr(torch.cuda, 'graph', graph)
    monkeypatch.setattr(torch.cuda, 'CUDAGraph', lambda: object())
    monkeypatch.setattr(torch.cuda, 'Stream', _Stream)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *a: _Stream())
    monkeypatch.setattr(torch.cuda, 'stream', lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, 'synchronize', lambda *a: None)
    monkeypatch.setattr(torch.cuda, 'graph_pool_handle', lambda: (0, 0))
    return state


def test_nothing_is_collected_inside_a_capture(fake_runtime):
    """Garbage with a finalizer, and a thread beside that allocates: no finalizer runs between a capture's begin and its end, and the
    collector is as it was afterwards, on again or off."""
    from speech2affective_gestures_amd import processor_v2 as P
    ends = []

    class Cycle:
        def __init__(self):
            self.me = self

        def __del__(self):
            ends.append((fake_runtime.inside, threading.current_thread().name))

    def allocate():
        return [[[] for _ in range(200)] for _ in range(200)]

    def segment():
        if not fake_runtime.inside:
            return
        Cycle()
        allocate()
        th = threading.Thread(target=allocate, name='beside')
        th.start()
        th.join()
    before = gc.isenabled(), gc.get_threshold()
    try:
        gc.set_threshold(50, 1, 1)
        for on in (True, False):
            (gc.enable if on else gc.disable)()
            P._GraphSegments([segment, segment], [None, None])
            assert gc.isenabled() == on
        gc.collect()
    finally:
        gc.set_threshold(*before[1])
        (gc.enable if before[0] else gc.disable)()
    assert len(ends) == 4 and not any(inside for inside, _ in ends), ends


def test_a_capture_that_fails_turns_the_collector_on_again(fake_runtime):
    from speech2affective_gestures_amd import processor_v2 as P

    def segment():
        if fake_runtime.inside:
            raise RuntimeError('inside')
    assert gc.isenabled()
    with pytest.raises(RuntimeError, match='inside'):
        P._GraphSegments([segment], [None])
    assert gc.isenabled()
