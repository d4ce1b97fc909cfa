"""CPU checks of the Python operator layer: argument validation mirrors the
reference (ValueError for shapes, kernel.py:2811-2816), CPU tensors are
refused (there is no CPU fallback), and the identity cache key tracks the
reference's discipline (kernel.py:2746-2748)."""
import pytest
import torch

import ratchet_b200 as rb
from ratchet_b200 import ops


def _mx_args(m_total=448, n=256, k=512, g=2, device="cpu"):
    return (torch.zeros((m_total, k), dtype=torch.float8_e4m3fn, device=device),
            torch.ones((m_total, k // 128), device=device),
            torch.zeros((g, n, k // 2), dtype=torch.uint8, device=device),
            torch.ones((g, n, k // 32), device=device),
            torch.zeros((m_total,), dtype=torch.int32, device=device))


def test_mx_rejects_n_not_multiple_of_128():
    a, asf, b, bsf, mi = _mx_args(n=200)
    with pytest.raises(ValueError, match="BLOCK_N"):
        rb.fp4_grouped_gemm(a, asf, b, bsf, mi)


def test_mx_rejects_k_not_multiple_of_128():
    a, asf, b, bsf, mi = _mx_args(k=192)
    with pytest.raises(ValueError, match="BLOCK_K"):
        rb.fp4_grouped_gemm(a, asf, b, bsf, mi)


def test_mx_rejects_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        rb.fp4_grouped_gemm(*_mx_args())


def test_mx_rejects_wrong_scale_dtype():
    a, asf, b, bsf, mi = _mx_args()
    with pytest.raises(ValueError, match="a_sf"):
        rb.fp4_grouped_gemm(a, asf.half(), b, bsf, mi)


def test_nvfp4_rejects_cpu_weights():
    b = [torch.zeros((256, 256), dtype=torch.uint8)]
    bsf = [torch.zeros((256, 32), dtype=torch.uint8)]
    with pytest.raises(ValueError, match="CUDA"):
        rb.pack_weights(b, bsf)


def test_nvfp4_rejects_mismatched_lists():
    with pytest.raises(ValueError):
        rb.nvfp4_grouped_gemm([], [], [], [])


def test_nvfp4_rejects_non_byte_dtype():
    with pytest.raises(ValueError, match="byte type"):
        ops._as_u8(torch.zeros(4, dtype=torch.float32), "x")


def test_identity_key_tracks_version_and_view():
    t = torch.zeros(8, dtype=torch.uint8)
    k0 = ops._identity(t)
    t.add_(1)                      # in-place write bumps _version
    assert ops._identity(t) != k0
    assert ops._identity(t[:4]) != ops._identity(t)


def test_lru_evicts_oldest():
    lru = ops._LRU()
    for i in range(ops._CACHE_MAX + 3):
        lru.get_or(i, lambda i=i: i)
    assert len(lru) == ops._CACHE_MAX
    assert 0 not in lru and (ops._CACHE_MAX + 2) in lru


def test_quantize_rejects_cpu():
    with pytest.raises(ValueError):
        rb.quantize_nvfp4(torch.zeros((4, 32)))


def test_problem_sizes_checked_against_tensors():
    """problem_sizes rows (M_g, N, K) must agree with the activation tensors;
    checked before any device work (a stand-in pack with no device buffer)."""
    import types

    fake = types.SimpleNamespace(n=256, k=128, device=torch.device("cpu"))
    a = [torch.zeros((m, 64), dtype=torch.uint8) for m in (3, 0, 17)]
    sf = [torch.zeros((m, 8), dtype=torch.uint8) for m in (3, 0, 17)]
    b = [None] * 3

    def call(ps):
        return rb.nvfp4_grouped_gemm(a, sf, b, b, ps, pack=fake)

    with pytest.raises(ValueError, match=r"problem_sizes\[0\]"):
        call([(4, 256, 128), (0, 256, 128), (17, 256, 128)])
    with pytest.raises(ValueError, match=r"problem_sizes\[0\]"):
        call(torch.tensor([[3, 128, 128], [0, 256, 128], [17, 256, 128]]))
    with pytest.raises(ValueError, match="3 groups"):
        call([(3, 256, 128)])
    # agreeing sizes pass the check and stop at the CPU tensors: no CPU fallback
    with pytest.raises(ValueError, match="CUDA"):
        call([(3, 256, 128), (0, 256, 128), (17, 256, 128)])
    with pytest.raises(ValueError, match=r"group 0: a \(3, 32\)"):
        rb.nvfp4_grouped_gemm([torch.zeros((3, 32), dtype=torch.uint8), a[1], a[2]], sf, b, b,
                              pack=fake)


def test_interleave_gate_up_order():
    """Rows come out as 16 gate rows, then the 16 up rows of the same outputs."""
    inter, k2 = 48, 4
    w = torch.arange(2 * inter, dtype=torch.uint8).view(-1, 1).repeat(1, k2)
    sf = w[:, :2].clone().view(torch.float8_e4m3fn)
    wi, sfi = rb.interleave_gate_up(w, sf)
    rows = wi[:, 0].tolist()
    want = []
    for c in range(inter // 16):
        want += list(range(16 * c, 16 * c + 16)) + list(range(inter + 16 * c, inter + 16 * c + 16))
    assert rows == want
    assert sfi.dtype == torch.float8_e4m3fn
    assert sfi.view(torch.uint8)[:, 0].tolist() == want
    with pytest.raises(ValueError):
        rb.interleave_gate_up(w[:40], sf[:40])


def test_last_status_is_the_calling_threads(monkeypatch):
    """Each thread's latest call; any thread's for one that made none; a call on another
    stream than the current one is waited for."""
    import contextlib
    import threading
    from types import SimpleNamespace

    from ratchet_b200 import _lib, ops

    read, waited = [], []
    fake = SimpleNamespace(fgg_read_device_status=lambda ws, stream: read.append((ws, stream)) or 0)
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    monkeypatch.setattr(ops, "_stream_ptr", lambda dev: 5)
    monkeypatch.setattr(ops.torch.cuda, "device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(ops.torch.cuda, "synchronize", waited.append)
    monkeypatch.setattr(ops, "_latest", None)
    monkeypatch.setattr(ops, "_LOCAL", ops._Local())
    call = lambda n, stream: ops._set_last_ws(SimpleNamespace(device="d", data_ptr=lambda: n), stream)

    def status(*made):
        out = []

        def work():
            for c in made:
                call(*c)
            ops.last_status()
            out.append((read.pop(), waited[:]))
            waited.clear()

        t = threading.Thread(target=work)
        t.start()
        t.join()
        return out[0]

    assert ops.last_status() == 0 and not read      # no call yet
    call(1, 5)
    assert status((2, 5)) == ((2, 5), [])
    ops.last_status()
    assert read.pop() == (1, 5) and not waited      # not the other thread's
    assert status((3, 5), (4, 7)) == ((4, 5), ["d"])
    assert status() == ((4, 5), ["d"])              # a thread without calls: the latest


def test_workspaces_are_kept_per_thread(monkeypatch):
    """Nine threads on one stream keep a workspace each, in every later call; a thread
    keeps those of eight streams."""
    import threading
    from types import SimpleNamespace

    from ratchet_b200 import ops

    monkeypatch.setattr(ops, "_capturing", None)
    monkeypatch.setattr(ops, "_LOCAL", ops._Local())
    monkeypatch.setattr(ops.torch, "empty", lambda n, **kw: SimpleNamespace(numel=lambda: n))
    dev = SimpleNamespace(index=0)
    threads = 9
    turn, kept = threading.Barrier(threads, timeout=30), [[] for _ in range(threads)]

    def work(i):
        for _ in range(3):
            turn.wait()
            kept[i].append(ops._workspace(dev, 11, 1000 + i))

    pool = [threading.Thread(target=work, args=(i,), daemon=True) for i in range(threads)]
    for t in pool:
        t.start()
    for t in pool:
        t.join(60)
    assert all(len(k) == 3 and k[0] is k[1] is k[2] for k in kept)
    assert len({id(k[0]) for k in kept}) == threads
    first = [ops._workspace(dev, s, 1000) for s in range(9)]
    assert all(ops._workspace(dev, s, 1000) is first[s] for s in range(1, 9))
    assert ops._workspace(dev, 0, 1000) is not first[0]
    assert ops._workspace(dev, 8, 2 << 20) is not first[8]      # too small


def test_threads_describe_their_own_problems(monkeypatch):
    """Two threads inside the NVFP4 entries at once, with the same geometry: each call's
    problem keeps its own pointers."""
    import threading
    from types import SimpleNamespace

    import torch

    from ratchet_b200 import _lib, ops

    both, got = threading.Barrier(2, timeout=30), {}

    def entry(prob, pack, ws, nbytes, stream):
        both.wait()          # the other thread has described its problem by now
        got[threading.current_thread().name] = (prob.a, prob.out)
        both.wait()
        return 0

    fake = SimpleNamespace(fgg_nvfp4_rows_workspace_bytes=lambda prob: 64,
                           fgg_nvfp4_grouped_gemm_rows=entry)
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    monkeypatch.setattr(ops, "_is_current", lambda dev: True)
    monkeypatch.setattr(ops, "_stream_ptr", lambda dev: 0)
    monkeypatch.setattr(ops, "_capturing", None)
    monkeypatch.setattr(ops, "_LOCAL", ops._Local())
    monkeypatch.setattr(ops, "_latest", None)
    cpu = torch.device("cpu")
    pack = SimpleNamespace(n=128, k=64, device=cpu, G=1, buf=torch.empty(1))
    off = torch.tensor([0, 4], dtype=torch.int32)
    want, scratch = {}, {}

    def work(name):
        a, sf = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8)
        out = torch.zeros(4, 128, dtype=torch.bfloat16)
        want[name] = (a.data_ptr(), out.data_ptr())
        scratch[name] = ops._scratch(3)
        ops.nvfp4_grouped_gemm_rows(a, sf, off, pack=pack, out=out)
        assert ops._scratch(3) is scratch[name]
        both.wait()          # the tensors live until both have been read

    pool = [threading.Thread(target=work, args=(n,), name=n, daemon=True) for n in ("x", "y")]
    for t in pool:
        t.start()
    for t in pool:
        t.join(60)
    assert len(got) == 2 and got == want
    assert scratch["x"][0] is not scratch["y"][0]
