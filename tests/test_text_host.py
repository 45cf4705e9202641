"""Text-model operators without a GPU: C ABI, refusals, and the kernels on the CPU device model."""
import ctypes as C
import os
import re
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, 'include', 's2ag_text.h')


@pytest.fixture(scope='module')
def lib():
    from speech2affective_gestures_amd import _lib, build
    build.build(force=False, verbose=False)
    return _lib.load()


def test_library_exports_the_text_operators(lib):
    from speech2affective_gestures_amd import _lib
    declared = set(re.findall(r'^(?:int|long long) (s2ag_\w+)\(', open(HEADER).read(), flags=re.M))
    assert declared == set(_lib.TEXT_SIGNATURES)
    for name in declared:
        assert hasattr(lib, name), name


def test_bound_structures_are_the_headers(tmp_path):
    """Sizes and offsets that a C compiler gives the header's structures against those of the binding."""
    from speech2affective_gestures_amd import _lib
    pairs = {'s2ag_clip_tensor': _lib.ClipTensor, 's2ag_lce_args': _lib.LceArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "s2ag_text.h"', 'int main(void) {']
    for name, cls in pairs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / 's.c'
    src.write_text('\n'.join(lines + ['return 0; }']))
    exe = str(tmp_path / 's')
    subprocess.check_call(['gcc', '-I' + os.path.join(ROOT, 'include'), str(src), '-o', exe])
    got = dict(ln.rsplit(' ', 1) for ln in subprocess.check_output([exe], text=True).splitlines())
    for name, cls in pairs.items():
        assert int(got[name]) == C.sizeof(cls)
        for f in cls._fields_:
            assert int(got[f'{name}.{f[0]}']) == getattr(cls, f[0]).offset, f


def test_entry_points_refuse_bad_arguments(lib):
    """Negative codes, nothing launched: null pointers, sizes beyond what is indexed, workspaces that are too small."""
    from speech2affective_gestures_amd import _lib
    BAD = -1
    p = C.c_void_p(4096)                                    # never read: every call below is refused
    assert lib.s2ag_emb_lookup(None, 0, p, 0, 4, 8, 10, 1.0, p, None) == BAD
    assert lib.s2ag_emb_lookup(p, 0, None, 0, 4, 8, 10, 1.0, p, None) == BAD
    assert lib.s2ag_emb_lookup(p, 0, p, 0, -1, 8, 10, 1.0, p, None) == BAD
    assert lib.s2ag_emb_lookup(p, 0, p, 0, 4, 0, 10, 1.0, p, None) == BAD
    assert lib.s2ag_emb_lookup(p, 0, p, 0, 4, 8, 0, 1.0, p, None) == BAD
    assert lib.s2ag_emb_lookup(p, 0, p, 0, 0, 8, 10, 1.0, p, None) == 0          # no ids: nothing to do
    for n, dim, entries in ((1 << 31, 8, 10), (4, 8, 1 << 30), (-1, 8, 10), (4, 1 << 25, 10)):
        assert lib.s2ag_emb_grad_workspace_bytes(n, dim, entries) == BAD
    need = lib.s2ag_emb_grad_workspace_bytes(100, 8, 10)
    assert need > 0
    grad = lambda ws=p, bytes_=need, ld=8, bf16=0, acc=0, dy=p: lib.s2ag_emb_grad(p, 0, dy, ld, bf16, 100, 8, 10, -1, 1.0, p, acc, ws, bytes_, None)  # noqa: E731
    assert grad(ws=None) == BAD and grad(bytes_=need - 1) == BAD and grad(ld=7) == BAD and grad(bf16=1, acc=1) == BAD and grad(dy=None) == BAD
    assert grad(ws=C.c_void_p(4097)) == BAD

    def args(**kw):
        a = _lib.LceArgs(x=4096, w=4096, target=4096, rows=10, vocab=20, ldx=8, ldw=8, dim=8, reduction=0, loss=4096, state=4096, workspace=4096,
                         workspace_bytes=1 << 40, grad_out=4096, dx=4096, dw=4096)
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    for kw in (dict(rows=-1), dict(rows=(1 << 21) + 1), dict(vocab=0), dict(vocab=(1 << 21) + 1), dict(dim=0), dict(ldx=7), dict(ldw=7), dict(reduction=3),
               dict(bf16=1, dw_accumulate=1)):
        a = args(**kw)
        assert lib.s2ag_lce_workspace_bytes(a, 0) == BAD and lib.s2ag_lce_state_bytes(a) == BAD, kw
        assert lib.s2ag_lce_fwd(a, None) == BAD and lib.s2ag_lce_bwd(a, None) == BAD, kw
    for kw in (dict(x=None), dict(w=None), dict(target=None), dict(state=None), dict(workspace=None), dict(workspace_bytes=64), dict(workspace=4100)):
        assert lib.s2ag_lce_fwd(args(**kw), None) == BAD, kw
        if kw != dict(target=None):
            assert lib.s2ag_lce_bwd(args(**kw), None) == BAD, kw
    assert lib.s2ag_lce_fwd(args(loss=None), None) == BAD and lib.s2ag_lce_bwd(args(grad_out=None), None) == BAD
    assert lib.s2ag_lce_bwd(args(dx=None, dw=None), None) == 0                    # no gradient is wanted

    t = (_lib.ClipTensor * 1)(_lib.ClipTensor(src=4096, dst=4096, n=10))
    assert lib.s2ag_clip_partials(t, 1) == 1 and lib.s2ag_clip_partials(t, -1) == BAD
    assert lib.s2ag_clip_grads(t, 1, 1.0, 0, None, p, None) == BAD and lib.s2ag_clip_grads(t, 1, 1.0, 0, p, None, None) == BAD
    assert lib.s2ag_clip_grads(t, 1, -1.0, 0, p, p, None) == BAD and lib.s2ag_clip_grads(t, 1, float('nan'), 0, p, p, None) == BAD
    for bad in (_lib.ClipTensor(src=4096, dst=4096, n=-1), _lib.ClipTensor(src=None, dst=4096, n=3), _lib.ClipTensor(src=4096, dst=4096, n=1 << 39),
                _lib.ClipTensor(src=4096, dst=4096, n=3, src_bf16=1)):
        assert lib.s2ag_clip_grads((_lib.ClipTensor * 1)(bad), 1, 1.0, 0, p, p, None) == BAD


def test_workspaces_cover_what_they_hold(lib):
    """The sizes that are asked for grow with what they must hold, at sizes where 32 bits would not do."""
    from speech2affective_gestures_amd import _lib
    n, dim, v = (1 << 31) - 65537, 2048, 131072
    tiles = -(-n // 64)
    assert lib.s2ag_emb_grad_workspace_bytes(n, dim, v) >= 4 * 4 * n + 4 * 2 * 2048 * tiles + v
    a = _lib.LceArgs(rows=1 << 21, vocab=1 << 21, ldx=4096, ldw=4096, dim=4096, bf16=0, dx=4096, dw=4096, keep=1)
    assert lib.s2ag_lce_state_bytes(a) >= 2 * 3 * 2 * (1 << 21) * 4096            # both operands in three pieces
    assert lib.s2ag_lce_workspace_bytes(a, 1) >= 4 * (1 << 21) * 4096 + 3 * 2 * (1 << 21) * 1024


def test_text_operators_refuse_cpu_tensors():
    if torch.cuda.is_available():
        pytest.skip('CPU tensors are refused before any GPU is asked for; checked where there is none')
    from speech2affective_gestures_amd import ops, optim
    ids, table = torch.zeros(3, dtype=torch.int64), torch.zeros(4, 5)
    with pytest.raises(RuntimeError, match='no CPU'):
        ops.embedding_sorted(ids, table)
    with pytest.raises(RuntimeError, match='no CPU'):
        ops.linear_cross_entropy(torch.zeros(3, 5), table, ids)
    with pytest.raises(RuntimeError, match='no CPU'):
        optim.clip_grads([table], 1.0)
    p = torch.nn.Parameter(table)
    p.grad = table.clone()
    with pytest.raises(RuntimeError, match='no CPU'):
        optim.clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError):
        optim.clip_grads([], 1.0)


# (-k expression, wavefront order, at least this many): a missing barrier changes results with the order
MODEL_RUNS = {'everything but the largest sums, in order': ('not case9 and not case10', 0, 200),
              'products and sorts, reversed order': ('cross_entropy and (case7 or case8 or reductions) or embedding_sorted and (case8 or case13 or case15)', 2, 20)}


@pytest.mark.parametrize('run', list(MODEL_RUNS))
def test_text_operators_on_the_cpu_device_model(run):
    expr, sched, at_least = MODEL_RUNS[run]
    env = dict(os.environ, S2AG_EMU='1', S2AG_EMU_SCHED=str(sched))
    env.pop('S2AG_HIP_LIB', None)
    cmd = [sys.executable, '-m', 'pytest', 'tests/test_gpu_text.py', '-m', 'gpu', '-q', '-p', 'no:cacheprovider', '-k', expr]
    p = subprocess.run(cmd, cwd=ROOT, env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=1500)
    m = re.search(r'(\d+) passed', p.stdout)
    assert p.returncode == 0 and m and int(m.group(1)) >= at_least, p.stdout[-3000:]
