"""CPU: the C-ABI shared library loads and exports every symbol include/ccnn.h declares."""
import os
import re

import gcn_amd.lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def declared_symbols():
    src = open(os.path.join(ROOT, "include", "ccnn.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    return sorted(set(re.findall(r"\b(ccnn_[a-z0-9_]+)\s*\(", src)))


def test_header_and_binding_agree():
    decl = declared_symbols()
    assert len(decl) >= 20
    assert sorted(L.EXPORTS) == decl


def test_library_exports_every_declared_symbol():
    lib = L.load()
    for name in declared_symbols():
        assert getattr(lib, name) is not None


def test_host_only_entry_points_work_without_gpu():
    d = L.dims(176)
    assert (d.re, d.mre, d.pout, d.nparams) == (79, 40, 800, 84853)
    assert d.off_b2 + 13 == d.nparams
    assert "workspace" in L.error_string(-2)
    lib = L.load()
    assert lib.ccnn_mbgd_workspace_bytes(128, 200, 4) > 0
    assert lib.ccnn_forward_workspace_bytes(10, 103, 8) > 0
    assert lib.ccnn_sgd_workspace_bytes(176) > 0
    assert lib.ccnn_mbgd_workspace_bytes(128, 5, 4) == 0      # too few bands
    try:
        L.dims(5)
        raise AssertionError("expected CcnnError")
    except L.CcnnError as e:
        assert e.code == -1


def test_step_path_choice_needs_no_gpu(monkeypatch):
    """ccnn_mbgd_path and the workspace size that follows it depend on the batch, the geometry and
    the element size only (never on a device), and CCNN_MBGD_PATH overrides the choice."""
    lib = L.load()
    monkeypatch.delenv("CCNN_MBGD_PATH", raising=False)
    assert lib.ccnn_mbgd_path(128, 103, 4) == 0            # the reference's batch sizes: one workgroup per sample
    assert lib.ccnn_mbgd_path(2048, 103, 4) == 1           # large batches: a tile of samples per workgroup
    assert lib.ccnn_mbgd_path(512, 103, 4) == 0 and lib.ccnn_mbgd_path(600, 103, 4) == 1
    assert lib.ccnn_mbgd_path(512, 200, 4) == 0 and lib.ccnn_mbgd_path(600, 200, 4) == 1
    assert lib.ccnn_mbgd_path(256, 176, 8) == 0 and lib.ccnn_mbgd_path(300, 176, 8) == 1
    assert lib.ccnn_mbgd_path(2048, 448, 8) == 2           # no tile fits the LDS: one launch per layer
    assert lib.ccnn_mbgd_path(0, 103, 4) < 0 and lib.ccnn_mbgd_path(128, 103, 2) < 0
    fused = lib.ccnn_mbgd_workspace_bytes(2048, 103, 4)
    monkeypatch.setenv("CCNN_MBGD_PATH", "fused")
    assert lib.ccnn_mbgd_path(2048, 103, 4) == 0
    assert lib.ccnn_mbgd_workspace_bytes(2048, 103, 4) > fused    # a conv-gradient row per sample, not per tile
    monkeypatch.setenv("CCNN_MBGD_PATH", "layers")
    assert lib.ccnn_mbgd_path(128, 103, 4) == 2


def test_tile_plans_fit_the_lds_for_every_geometry():
    """tile_plan (the host-side choice of waves, samples per tile and delta-image chunks of the
    sample-tile kernel) never asks for more LDS than a workgroup may have, covers the batch, and
    keeps one sample per wave - for every band count and both element sizes."""
    import ctypes as C

    class Plan(C.Structure):
        _fields_ = [("nwv", C.c_int), ("ms", C.c_int), ("nch", C.c_int), ("smem", C.c_size_t), ("tiles", C.c_int)]

    lib = L.load()
    fits = 0
    for es, sym in ((4, "_ZN4ccnn9tile_planIfEEbiRK9ccnn_dimsPNS_8TilePlanE"), (8, "_ZN4ccnn9tile_planIdEEbiRK9ccnn_dimsPNS_8TilePlanE")):
        fn = getattr(lib, sym)
        fn.restype = C.c_bool
        for z in range(21, 449):
            d = L.dims(z)
            for B in (1, 7, 256, 600, 2048, 5000):
                p = Plan()
                if not fn(B, C.byref(d), C.byref(p)):
                    assert lib.ccnn_mbgd_path(B, z, es) != 1      # no tile: the library must not pick that path
                    continue
                fits += 1
                assert p.smem <= 160 * 1024, (z, B, es, p.smem)
                assert p.nwv in (4, 8, 16) and 1 <= p.ms <= min(p.nwv, 8) and p.nch in (1, 2, 4, 8)
                assert p.tiles == (B + p.ms - 1) // p.ms
    assert fits > 3000


def test_integration_sketch_compiles_against_the_header(tmp_path):
    """Every ```cpp block of INTEGRATION.md that includes <ccnn.h> is compiled (-fsyntax-only) against
    include/ccnn.h: the document a maintainer copies from cannot drift from the boundary it describes."""
    import shutil
    import subprocess
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    blocks = [b for b in re.findall(r"```cpp\n(.*?)```", text, flags=re.S) if "#include <ccnn.h>" in b]
    assert blocks, "INTEGRATION.md lost its compilable sketch"
    cxx = shutil.which("g++") or "g++"     # host code only: the sketch is what a plain C++ trainer would hold
    for i, b in enumerate(blocks):
        src = tmp_path / f"sketch{i}.cpp"
        src.write_text(b)
        r = subprocess.run([cxx, "-std=c++17", "-fsyntax-only", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__",
                            "-I", "/opt/rocm/include", "-I", os.path.join(ROOT, "include"), str(src)],
                           capture_output=True, text=True)
        assert r.returncode == 0, r.stderr


def test_scoring_and_optimiser_calls_refuse_bad_arguments():
    """The argument checks of ccnn_log_probs*, ccnn_grad_norm and ccnn_adamw_* answer before anything is launched."""
    import ctypes as C
    lib, ok, nul = L.load(), C.c_void_p(64), C.c_void_p()

    def score(x=ok, kind=1, rows=2, classes=5, stride=5, y=ok, yb=4, top=2, tl=ok, ti=ok, stats=ok):
        return lib.ccnn_log_probs(x, kind, rows, classes, stride, y, yb, top, 1, stats, tl, ti, nul, 0, nul)

    assert score(rows=0) == 0
    for bad in (dict(x=nul), dict(kind=0), dict(kind=5), dict(rows=-1), dict(classes=0), dict(stride=4), dict(y=nul),
                dict(yb=2), dict(top=-1), dict(top=6), dict(tl=nul), dict(ti=nul), dict(stats=nul)):
        assert score(**bad) == -1, bad
    assert score(rows=1 << 31) == -3 and score(classes=(1 << 30) + 1, stride=1 << 40) == -3
    assert score(classes=100, stride=100, top=65) == -1

    def grad(x=ok, kind=1, classes=5, stride=5, stats=ok, dl=ok, dh=ok, out=C.c_void_p(4096), ostride=5, rows=2):
        return lib.ccnn_log_probs_grad(x, kind, rows, classes, stride, ok, 4, stats, dl, dh, out, ostride, nul)

    assert grad(rows=0) == 0
    for bad in (dict(x=nul), dict(kind=9), dict(stats=nul), dict(dl=nul, dh=nul), dict(out=nul), dict(ostride=4),
                dict(out=ok, ostride=6)):
        assert grad(**bad) == -1, bad

    def norm(at=(64, 64), n=(10, 400000), kinds=(1, 3), limit=1.0, out=ok, ws=ok, short=0, count=None):
        c = len(at)
        n = (C.c_long * c)(*n)
        need = lib.ccnn_grad_norm_workspace_bytes(n, c)
        assert need >= 8 or n[0] < 0 or n[1] < 9000
        return lib.ccnn_grad_norm((C.c_void_p * c)(*at), n, (C.c_int * c)(*kinds), c if count is None else count, limit, out, ws,
                                  need - short, nul)

    assert norm(short=1) == -2 and norm(ws=nul) == -2
    for bad in (dict(limit=0.0), dict(limit=float("nan")), dict(out=nul), dict(count=-1), dict(at=(0, 64)), dict(n=(-1, 5)),
                dict(kinds=(1, 7)), dict(kinds=(0, 1))):
        assert norm(**bad) == -1, bad

    fine = (64, 10, 0, 0, 0.1, 1)

    def step(*ts, grads=None, kinds=None, bits=32, m=ok, v=ok, ms=ok, vs=ok, master=ok, clock=ok, b1=0.9, b2=0.999, eps=1e-8):
        k = max(1, len(ts))
        arr = (L.AdamwTensor * k)(*ts)
        return lib.ccnn_adamw_step(arr, (C.c_void_p * k)(*(grads or [64] * k)), (C.c_int * k)(*(kinds or [t[5] for t in ts])),
                                   len(ts), bits, m, v, ms, vs, master, clock, 1e-3, nul, b1, b2, eps, nul, nul)

    for bad in (dict(bits=16), dict(m=nul), dict(v=nul), dict(clock=nul), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0),
                dict(bits=8, ms=nul), dict(bits=8, vs=nul), dict(b1=float("nan")), dict(grads=[0]), dict(kinds=[3])):
        assert step(fine, **bad) == -1, bad
    assert step((64, 10, 0, 0, 0.1, 3), master=nul) == -1                  # half precision without its master copy
    assert step((64, 10, 0, 0, 0.1, 2), bits=8) == -1                      # 8-bit moments of doubles
    assert step(fine, (64, 10, 0, 0, 0.1, 2)) == -1                        # doubles among others
    assert step((64, 10, 0, 0, 0.1, 3), kinds=[4]) == -1
    assert step(fine, eps=0.0) == -1 and step(fine, eps=1e-46) == -1 and step((64, 10, 0, 0, 0.1, 2), eps=0.0) == -1
    for bad in ((0, 10, 0, 0, 0.1, 1), (64, -1, 0, 0, 0.1, 1), (64, 10, -1, 0, 0.1, 1), (64, 10, 0, -1, 0.1, 1),
                (64, 10, 0, 0, 0.1, 0)):
        assert step(bad) == -1, bad
    arr = (L.AdamwTensor * 1)(fine)
    assert lib.ccnn_adamw_moments(arr, 1, nul, ok, ok, ok, ok, ok, nul) == -1
    assert lib.ccnn_adamw_moments(arr, -1, ok, ok, ok, ok, ok, ok, nul) == -1
