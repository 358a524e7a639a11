"""Refusals of the faces of a step behind a shared prefix that go by sizes and places alone: on the host, with nothing launched."""
import types

import pytest
import torch

from janus_b200.kernels import ops


@pytest.fixture
def launches(monkeypatch):
    """The entry points' calls, which do nothing."""
    calls = []

    def entry(name):
        return lambda *args: (calls.append(name), 0)[1]
    names = ("jb_step_tables", "jb_attention_prefix_f32", "jb_attention_prefix_bf16", "jb_verify_drafts")
    monkeypatch.setattr(ops, "_lib", lambda *args: types.SimpleNamespace(**{n: entry(n) for n in names}))
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "kernel_status", lambda device: torch.zeros(1, dtype=torch.int32))
    with ops.unchecked():           # (the checks of tensors want a device)
        yield calls


@pytest.fixture
def refused(monkeypatch):
    """The library itself, on tensors of the host: only calls that it refuses before a launch."""
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    with ops.unchecked():
        yield


INPUTS = ("lengths", "new_tokens", "rows", "old_table", "old_held", "prefix_pages", "old_free", "old_n_free")


def tables_tensors(B=5, B0=4, W0=6, W=8, P=2, N=30, T=40):
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32)      # noqa: E731
    return dict(lengths=z(B), new_tokens=z(B), rows=z(B), old_table=z(B0, W0), old_held=z(B0), prefix_pages=z(P), old_free=z(N), old_n_free=z(1),
                q_start=z(B + 1), kv_len=z(B), positions=z(T), token_seq=z(T), dest_rows=z(T), table=z(B, W), held=z(B), free_pages=z(N),
                n_free=z(1), missing=z(1))


def run_tables(t):
    ops.step_tables(*(t[n] for n in INPUTS), **{n: v for n, v in t.items() if n not in INPUTS}, page_size=64)


def laid_over(t, first, second, shift):
    """`first` and `second` as views of one tensor, the second `shift` numbers behind the first's begin."""
    n, m = t[first].numel(), t[second].numel()
    low = min(0, shift)
    both = torch.zeros(max(n, shift + m) - low, dtype=torch.int32)
    return {**t, first: both[-low:n - low].view(t[first].shape), second: both[shift - low:shift - low + m].view(t[second].shape)}


@pytest.mark.parametrize("made", ["q_start", "table", "free_pages", "n_free"])
@pytest.mark.parametrize("given", ["lengths", "old_table", "old_free", "old_n_free"])
def test_tables_are_not_made_over_what_they_are_made_from(refused, given, made):
    t = tables_tensors()
    n, m = t[given].numel(), t[made].numel()
    for shift in {0, n - 1, 1 - m, n // 2, -(m // 2)}:
        with pytest.raises(ops.KernelError, match="cannot lie"):
            run_tables(laid_over(t, given, made, shift))


@pytest.mark.parametrize("first,second,shift", [("positions", "dest_rows", 39), ("dest_rows", "positions", -39), ("held", "missing", 4), ("table", "table", 0)])
def test_tables_are_not_made_over_each_other(refused, first, second, shift):
    t = tables_tensors()
    t = laid_over(t, first, second, shift) if first != second else {**t, "token_seq": t["table"].view(-1)}
    with pytest.raises(ops.KernelError, match="each other"):
        run_tables(t)


@pytest.mark.gpu
def test_tables_side_by_side_and_inputs_that_share_a_place():
    want = {k: v.cpu() for k, v in run_on_device(tables_tensors()).items()}
    t = tables_tensors()
    for given in ("lengths", "old_table", "old_free", "old_n_free"):
        for made in ("q_start", "table", "free_pages", "n_free"):
            for shift in (t[given].numel(), -t[made].numel()):
                got = run_on_device(laid_over(t, given, made, shift))
                assert all(torch.equal(want[k], got[k].cpu()) for k in want)
    run_on_device(laid_over(t, "lengths", "old_table", 1))
    run_on_device({**t, "new_tokens": t["lengths"]})
    run_on_device(tables_tensors(B0=0, P=0, T=0))
    everything = torch.zeros(sum(v.numel() for v in t.values()), dtype=torch.int32)
    run_on_device({k: piece.view(v.shape) for (k, v), piece in zip(t.items(), everything.split([v.numel() for v in t.values()]))})
    torch.cuda.synchronize()


def run_on_device(t):
    """The call on the device, tensors that share a storage sharing one there; the outputs."""
    storages = {v.untyped_storage().data_ptr(): v for v in t.values() if v.numel()}
    moved = {p: torch.zeros(v.untyped_storage().nbytes() // 4, dtype=torch.int32, device="cuda") for p, v in storages.items()}
    there = {k: moved[v.untyped_storage().data_ptr()].as_strided(v.shape, v.stride(), v.storage_offset()) if v.numel() else v.cuda()
             for k, v in t.items()}
    run_tables(there)
    return {k: v for k, v in there.items() if k not in INPUTS}


def run_attention(dtype=torch.bfloat16, nh=8, nkv=2, hd=64, T=3, n=2):
    z = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype)      # noqa: E731
    from janus_b200.engine.workspace import Workspace
    ops.attention_prefix(z(T, nh * hd, dtype=dtype), z(4, max(nkv, 0), 64, hd, dtype=dtype), z(4, max(nkv, 0), 64, hd, dtype=dtype),
                         z(T, nh * hd, dtype=dtype), z(1), 64, z(n, 1), z(n + 1), z(n), z(T), nh, nkv, hd, 64, 0.125,
                         Workspace(torch.device("cpu")), 2, 128)


@pytest.mark.parametrize("dtype,nh,nkv,hd", [
    (torch.bfloat16, 129, 1, 64), (torch.bfloat16, 516, 4, 64), (torch.bfloat16, 2, 4, 64), (torch.bfloat16, 6, 4, 64), (torch.bfloat16, 8, 0, 64),
    (torch.float32, 2, 4, 64), (torch.float32, 7, 2, 64), (torch.float32, 8, 0, 64), (torch.float32, 4, 2, 257), (torch.bfloat16, 4, 2, 264)])
def test_attention_refuses_heads_that_it_does_not_take(launches, dtype, nh, nkv, hd):
    with pytest.raises(ops.KernelError, match="attention_prefix"):
        run_attention(dtype, nh, nkv, hd)
    assert not launches


@pytest.mark.parametrize("dtype,nh,nkv,hd", [(torch.bfloat16, 128, 1, 64), (torch.bfloat16, 7, 7, 256), (torch.float32, 129, 1, 37), (torch.float32, 8, 4, 256)])
def test_attention_takes_the_heads_at_its_limits(launches, dtype, nh, nkv, hd):
    run_attention(dtype, nh, nkv, hd)
    assert len(launches) == 1


@pytest.mark.parametrize("name", ["_cuda_getCurrentRawStream", "_cuda_getDevice"])
def test_the_current_stream_is_found_without_names_of_torchs_own(name):
    """A torch that lacks them (one without CUDA, a later one) still imports the library, and the public way answers."""
    import os
    import subprocess
    import sys
    code = (f"import types, torch\ndel torch._C.{name}\nimport janus_b200.kernels.ops as ops\n"
            "torch.cuda.current_stream = lambda: types.SimpleNamespace(cuda_stream=1234)\nassert ops._stream() == 1234")
    root = os.path.dirname(os.path.dirname(os.path.abspath(ops.__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(root), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
