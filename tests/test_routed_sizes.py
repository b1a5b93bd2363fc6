"""Sizes that the Python entries of the routed steps refuse, without a GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

FAR = (1 << 32) + 4  # 4 once cut to 32 bits


def wide(rows, cols, dtype=torch.float32):
    """A matrix of these sizes over one element."""
    return torch.zeros(1, 1, dtype=dtype).expand(rows, cols)


@pytest.fixture
def lib(monkeypatch):
    import build as mvbuild
    mvbuild.build()
    import mvllm_moe
    # Host tensors pass for the library's device; no entry is reached.
    monkeypatch.setattr(mvllm_moe, "_device", -1)
    monkeypatch.setattr(mvllm_moe, "_stream_at", lambda stream, t: None)

    def reached(rc):
        raise AssertionError("the C entry was called")

    monkeypatch.setattr(mvllm_moe, "_check", reached)
    return mvllm_moe


def test_sizes_past_32_bits_are_refused(lib):
    i32 = torch.int32
    pos, x, rw = torch.zeros(4, 2, dtype=i32), torch.zeros(4, 8), torch.zeros(8)
    far_pos, far_rows, far_cols = wide(FAR, 2, i32), wide(FAR, 8), wide(4, FAR)
    dwt = torch.zeros(4, 2)
    fmt, w, s = lib.FMT_INT4_G64, torch.zeros(64, dtype=torch.uint8), torch.zeros(64)
    nr, tab = torch.zeros(2, dtype=i32), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: lib.dispatch_dev(far_cols, pos, far_cols),
                 lambda: lib.dispatch_dev(x, pos, far_rows),
                 lambda: lib.dispatch_dev(far_rows, far_pos, x),
                 lambda: lib.dispatch_grad_dev(far_rows, pos, x),
                 lambda: lib.combine_dev(far_rows, rw, pos, x),
                 lambda: lib.combine_dev(far_cols, rw, pos, far_cols),
                 lambda: lib.combine_grad_dev(x, far_rows, rw, pos, pos, far_rows, dwt),
                 lambda: lib.route_grad_dev(x, wide(FAR, 8), pos, wide(4, FAR), dwt, nr, nr, nr,
                                            pos, x, None, workspace=x),
                 lambda: lib.matvec_q4_dev(fmt, far_rows, w, s, far_rows),
                 lambda: lib.matvec_q4_dev(fmt, far_cols, w, s, x),
                 lambda: lib.matvec_q4_grad_dev(fmt, x, w, s, far_cols),
                 lambda: lib.expert_matvec_q4_dev(fmt, far_rows, tab, tab, nr, nr, far_rows),
                 lambda: lib.expert_matvec_q4_grad_dev(fmt, x, tab, tab, nr, nr, far_cols)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()


def test_missing_tensors_are_named(lib):
    i32 = torch.int32
    pos, x, rw, dwt = torch.zeros(4, 2, dtype=i32), torch.zeros(4, 8), torch.zeros(8), wide(4, 2)
    nr, tab = torch.zeros(2, dtype=i32), torch.zeros(2, dtype=torch.int64)
    router, scores, args = torch.zeros(2, 8), torch.zeros(4, 2), (nr, nr, nr)
    for name, call in (
            ("tok_pos", lambda: lib.dispatch_dev(x, None, x)),
            ("dwt", lambda: lib.combine_grad_dev(x, x, rw, pos, pos, x, None)),
            ("scores", lambda: lib.route_grad_dev(x, router, pos, None, dwt, *args, pos, x, None,
                                                  workspace=x)),
            ("nr", lambda: lib.expert_matvec_q4_dev(lib.FMT_INT4_G64, x, tab, tab, None, nr, x))):
        with pytest.raises(ValueError, match=name):
            call()


def test_plans_refuse_what_the_products_refuse(lib):
    plan = (ctypes.c_int * 8)()
    good = [lib.FMT_INT4_G64, 0, lib.DTYPE_F32, 1, 2, 64, 64, plan]
    entry = lib.lib().mvllm_matvec_q4_plan
    if not lib.available():
        assert entry(*good) == lib.ERR_NOT_INIT
    for at, bad in ((0, 0), (0, 8), (2, 7), (3, 0), (3, 1025), (4, 0), (4, (1 << 30) + 1), (5, 0),
                    (6, (1 << 30) + 1), (7, None)):
        args = list(good)
        args[at] = bad
        assert entry(*args) == lib.ERR_INVALID, at
