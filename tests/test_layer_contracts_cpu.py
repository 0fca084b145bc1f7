"""Refusals of the layer operators' C entry points where operands share memory, before any launch: runs without a GPU."""
import ctypes as C

BASE = 0x7f0000000000      # addresses that nothing reads: every call below is refused first


def at(i, off=0):
    return C.c_void_p(BASE + i * 0x1000000 + off)


def _err(lib):
    return lib.ssd_last_error().decode()


def test_step_outputs_that_share_memory_are_refused(lib):
    """selscan step and conv1d step: y / out over the state, the history or operands that other threads read; the state or the history over
    an operand.  Rows that lie between one another share nothing; the operand itself may be the output (both on the GPU's tests)."""
    from trading_bot_0_b200 import _lib as L
    S, D, N = 4, 48, 16
    s = L.SsdSelStepDims()
    s.streams, s.channels, s.dstate, s.ngroups, s.dtype, s.device = S, D, N, 1, L.SSD_BF16, -1
    names = ("state", "x", "dt", "A", "Bm", "Cm", "D", "z", "y", "dt_bias")

    def call(**kw):
        q = L.SsdStepPtrs()
        for i, n in enumerate(names):
            setattr(q, n, kw.get(n, at(i + 1)))
        return lib.ssd_selscan_step(C.byref(s), C.byref(q), None)
    row = D * 2
    where = {n: i + 1 for i, n in enumerate(names)}
    for n in ("state", "A", "Bm", "Cm", "D", "dt_bias"):
        assert call(y=at(where[n])) == -1 and "share" in _err(lib), n
    for n in ("x", "dt", "z"):                            # rows moved against the operand's own
        for off in (2, -2, row, -row, (S - 1) * row):
            assert call(y=at(where[n], off)) == -1 and "share" in _err(lib), (n, off)
    for n in names[1:]:
        if n != "y":
            assert call(**{n: at(1, 64)}) == -1 and "state" in _err(lib), n
    s.x_stride_s, s.y_stride_s = 100, 100                 # rows 100 apart, the output's beginning inside the operand's
    for off in (2 * 47, -2 * 47, 200 - 2 * 47, 3 * 200 + 2):
        assert call(y=at(where["x"], off)) == -1 and "share" in _err(lib), off
    s.y_stride_s = 150                                    # other rows: anything inside the operand's bytes
    assert call(y=at(where["x"])) == -1

    d = L.SsdConvDims()
    d.batch, d.seqlen, d.channels, d.width, d.dtype, d.device, d.activation = S, 1, 64, 4, L.SSD_BF16, -1, 1
    d.in_stride_l = d.out_stride_l = d.in_stride_b = d.out_stride_b = 64
    step = lambda x, w, b, h, o: lib.ssd_conv1d_step(C.byref(d), x, w, b, h, o, None)
    for a in ((at(1), at(2), None, at(4), at(4)), (at(1), at(2), None, at(4), at(4, 1024)), (at(1), at(2), None, at(4), at(1, 128)),
              (at(1), at(2), None, at(4), at(1, -128)), (at(1), at(2), None, at(4), at(2)), (at(1), at(2), at(3), at(4), at(3)),
              (at(4, 256), at(2), None, at(4), at(5)), (at(1), at(4), None, at(4), at(5)), (at(1), at(2), at(4, 512), at(4), at(5))):
        assert step(*a) == -1 and "share" in _err(lib), a


def test_projection_workspaces_start_on_a_word(lib):
    from trading_bot_0_b200 import _lib as L
    d = L.SsdLinearDims()
    d.rows, d.in_features, d.out_features, d.dtype, d.device = 100, 64, 96, L.SSD_BF16, -1
    fwd, bwd = (lib.ssd_linear_workspace_bytes(C.byref(d), p) for p in (0, 1))
    assert lib.ssd_linear_forward(C.byref(d), at(1), at(2), None, None, at(3), None, at(9, 2), fwd, None) == -2 and "4-byte" in _err(lib)
    assert lib.ssd_linear_backward(C.byref(d), at(1), at(2), None, at(3), 0, at(4), at(5), None, at(9, 1), bwd, None) == -2 and "4-byte" in _err(lib)
