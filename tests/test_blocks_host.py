"""CPU tests of the 8-bit linear path (RMSNormalization, QuantizeBlocks,
MatMulBlockScaled): what the C entries and the operator classes refuse, the
layouts the classes read and write, shapes and registration.  No kernel runs:
the C entries check their arguments before they look at the (null) handle."""
import ctypes

import pytest
import torch

F32, F16, BF16, E4M3 = 0, 1, 2, 3


@pytest.fixture(scope="module")
def C(ob):
    return ob._capi


def norm_desc(C, **kw):
    d = C.RmsNormDesc(rows=4, cols=256, type=BF16, weight_type=BF16, out_type=BF16, epsilon=1e-5)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def quant_desc(C, **kw):
    d = C.QuantizeDesc(rows=4, cols=256, type=BF16, block_rows=1)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def mm_desc(C, **kw):
    d = C.MatmulBlocksDesc(m=4, n=256, k=256, out_type=F32)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


P = ctypes.c_void_p(4096)  # never read


def call_norm(C, d, x=P, res=None, w=P, s=None, y=P, ys=P):
    return C.lib().onnxb200_rmsnorm(None, ctypes.byref(d) if d else None, x, res, w, s, y, ys)


def call_quant(C, d, x=P, q=P, s=P):
    return C.lib().onnxb200_quantize_blocks(None, ctypes.byref(d) if d else None, x, q, s)


def call_mm(C, d, a=P, sa=P, b=P, sb=P, bias=None, y=P):
    return C.lib().onnxb200_matmul_blocks(None, ctypes.byref(d) if d else None, a, sa, b, sb, bias, y)


def test_valid_arguments_reach_the_handle_check(C):
    odd = ctypes.c_void_p(4097)
    for rc in (call_norm(C, norm_desc(C)), call_norm(C, norm_desc(C, out_type=E4M3)), call_quant(C, quant_desc(C)),
               call_quant(C, quant_desc(C, block_rows=128)), call_mm(C, mm_desc(C)), call_mm(C, mm_desc(C, k=0), None, None, None, None),
               call_norm(C, norm_desc(C, rows=0), None, None, None, None, None, None),
               call_quant(C, quant_desc(C, cols=0), None, None, None), call_mm(C, mm_desc(C, m=0), None, None, None, None),
               call_mm(C, mm_desc(C, a_scale_row=0, a_scale_block=1)),  # one row of scales for all rows of a
               call_mm(C, mm_desc(C, lda=257), a=odd),                  # bytes have no alignment of their own
               call_norm(C, norm_desc(C, cols=C.RMSNORM_MAX_COLS))):
        assert rc == C.ERR_INVALID_ARGUMENT
    # the null descriptor and the null handle give the same code; the others below do not
    assert call_norm(C, None) == call_quant(C, None) == call_mm(C, None) == C.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("kw", [
    {"type": E4M3}, {"type": 7}, {"type": -1}, {"weight_type": E4M3}, {"out_type": F32}, {"out_type": F16},
    {"rows": -1}, {"rows": 1 << 31}, {"cols": 0}, {"cols": -5}, {"epsilon": -1.0}, {"epsilon": float("nan")},
    {"ldx": 255}, {"ldr": 1}, {"lds": -256}, {"ldy": 128}, {"ldx": 1 << 40},
    {"out_type": E4M3, "y_scale_row": 1, "y_scale_block": 1}, {"out_type": E4M3, "y_scale_row": 1, "y_scale_block": 3},
    {"out_type": E4M3, "y_scale_row": 0, "y_scale_block": 1}, {"out_type": E4M3, "y_scale_row": -2, "y_scale_block": 1},
])
def test_rmsnorm_refuses(C, kw):
    assert call_norm(C, norm_desc(C, **kw)) == C.ERR_VALIDATION


def test_rmsnorm_refuses_long_rows_and_bad_pointers(C):
    assert call_norm(C, norm_desc(C, cols=C.RMSNORM_MAX_COLS + 1)) == C.ERR_UNSUPPORTED
    odd = ctypes.c_void_p(4097)
    assert call_norm(C, norm_desc(C), x=odd) == C.ERR_VALIDATION
    assert call_norm(C, norm_desc(C), res=odd) == C.ERR_VALIDATION
    assert call_norm(C, norm_desc(C), s=odd) == C.ERR_VALIDATION
    assert call_norm(C, norm_desc(C), w=odd) == C.ERR_VALIDATION
    assert call_norm(C, norm_desc(C), y=odd) == C.ERR_VALIDATION
    assert call_norm(C, norm_desc(C, out_type=E4M3), y=odd, ys=odd) == C.ERR_VALIDATION


@pytest.mark.parametrize("kw", [
    {"type": E4M3}, {"type": 9}, {"block_rows": 0}, {"block_rows": 64}, {"rows": -1}, {"cols": -1}, {"cols": 1 << 31},
    {"ldx": 255}, {"ldq": 17}, {"scale_row": 1, "scale_block": 1}, {"scale_row": 1, "scale_block": 0},
    {"rows": 300, "block_rows": 128, "scale_row": 1, "scale_block": 2},
])
def test_quantize_refuses(C, kw):
    assert call_quant(C, quant_desc(C, **kw)) == C.ERR_VALIDATION


def test_quantize_refuses_too_many_blocks_and_bad_pointers(C):
    assert call_quant(C, quant_desc(C, rows=1 << 30, cols=1024)) == C.ERR_UNSUPPORTED
    assert call_quant(C, quant_desc(C), x=ctypes.c_void_p(4097)) == C.ERR_VALIDATION
    assert call_quant(C, quant_desc(C), s=ctypes.c_void_p(4098)) == C.ERR_VALIDATION


@pytest.mark.parametrize("kw", [
    {"out_type": E4M3}, {"out_type": 4}, {"flags": 1}, {"flags": 16}, {"m": -1}, {"n": -1}, {"k": -1}, {"m": 1 << 31},
    {"lda": 255}, {"ldb": -1}, {"ldy": 100}, {"a_scale_row": -1, "a_scale_block": 1}, {"b_scale_row": 1, "b_scale_block": -1},
])
def test_matmul_refuses(C, kw):
    assert call_mm(C, mm_desc(C, **kw)) == C.ERR_VALIDATION


def test_matmul_refuses_too_many_tiles_and_bad_pointers(C):
    assert call_mm(C, mm_desc(C, m=1 << 30, n=1 << 30)) == C.ERR_UNSUPPORTED
    odd = ctypes.c_void_p(4097)
    assert call_mm(C, mm_desc(C), sa=odd) == call_mm(C, mm_desc(C), sb=odd) == C.ERR_VALIDATION
    assert call_mm(C, mm_desc(C), bias=odd) == call_mm(C, mm_desc(C), y=odd) == C.ERR_VALIDATION


def test_row_stride(ob):
    stride = ob.ops._row_stride
    x = torch.zeros(6, 40)
    assert stride(x, "x") == 40
    assert stride(x[:, :33], "x") == 40
    assert stride(x[::2, :33], "x") == 80
    assert stride(torch.zeros(2, 3, 40)[:, :, :7], "x") == 40
    assert stride(torch.zeros(5), "x") == 5
    assert stride(torch.zeros(5, 0), "x") == 0
    assert stride(torch.zeros(4, 1)[::2], "x") == 2
    assert stride(x[:1, :33], "x") == 33  # a single row has no stride
    for bad in (x.t(), x[:, ::2], torch.zeros(2, 3, 40)[:, :2], torch.zeros(1, 40).expand(6, 40), torch.zeros(())):
        with pytest.raises(ob.ValidationError):
            stride(bad, "x")


def test_stored_layouts(ob):
    new = lambda spec: ob.ops._new_on(torch.device("cpu"))(*spec)
    q = new(ob.ops._stored_rows((3, 2), 33))
    assert q.shape == (3, 2, 33) and ob.ops._stored_stride(33) == 48 and ob.ops._row_stride(q, "q") == 48
    q = new(ob.ops._stored_rows((), 64))
    assert q.shape == (64,) and ob.ops._stored_stride(64) == 64
    for shape in ((), (4,), (3, 0), (0, 3), (2, 3, 4)):
        assert new(ob.ops._dense(shape, torch.float32)).stride() == torch.empty(shape).stride()
    for lead, rows in (((3, 2), 6), ((6,), 6), ((), 1), ((1,), 1), ((0,), 0)):
        s = new(ob.ops._stored_scales(lead, rows, 5))
        assert s.shape == (*lead, 5)
        back, sr, sb = ob.ops._scale_strides(s, rows, 5, "s")
        assert back.data_ptr() == s.data_ptr()  # read in place, never copied
        assert rows <= 1 or (sr, sb) == (1, rows)


def test_scale_strides(ob):
    f = ob.ops._scale_strides
    one = torch.ones(1, 1).expand(4, 3)  # one value for all: laid out densely
    s, sr, sb = f(one, 4, 3, "s")
    assert (sr, sb) == (3, 1) and s.is_contiguous()
    row = torch.ones(1, 3).expand(4, 3)  # one row for all rows: read as it is
    s, sr, sb = f(row, 4, 3, "s")
    assert (sr, sb) == (0, 1)
    for bad in (torch.ones(4, 4), torch.ones(3, 3), torch.ones(4, 3).double(), torch.tensor(1.0)):
        with pytest.raises(ob.ValidationError):
            f(bad, 4, 3, "s")


def test_operators_refuse_host_tensors_and_bad_arguments(ob):
    class NoGpu:
        device = 0
    ctx = ob.ExecutionContext(NoGpu())
    x = torch.zeros(2, 128)
    for call in (lambda: ob.RMSNormalization().compute([x, x[0]], ctx), lambda: ob.QuantizeBlocks().compute([x], ctx),
                 lambda: ob.MatMulBlockScaled().compute([x, x, x, x], ctx)):
        with pytest.raises(ob.ValidationError, match="expected tensors on cuda:0"):
            call()
    with pytest.raises(ob.ValidationError):
        ob.QuantizeBlocks(block_rows=64)
    with pytest.raises(ob.ValidationError):
        ob.MatMulBlockScaled(dtype=torch.float64)
    with pytest.raises(ob.UnsupportedFeature):
        ob.RMSNormalization(axis=1).output_shapes({"attrs": {"axis": 1}}, [[2, 3, 4]])


def test_registry_and_shapes(ob):
    r = ob.OperatorRegistry.initialize_standard_operators()
    node = {"op": "RMSNormalization", "inputs": ["x", "w"], "outputs": ["y"], "attrs": {"epsilon": 1e-6, "axis": -1}}
    op = r.create_operator_for_node(node, opset=23)
    assert isinstance(op, ob.RMSNormalization) and op.epsilon == 1e-6
    op.validate(node)
    assert op.output_shapes(node, [[2, 3, 128], [128]]) == [[2, 3, 128]]
    with pytest.raises(ob.InvalidOperator):  # not in the opset before 23
        r.create_operator_for_node(node, opset=22)
    qn = {"op": "QuantizeBlocks", "domain": "b200", "inputs": ["x"], "outputs": ["q", "s"], "attrs": {"block_rows": 128}}
    assert r.create_operator_for_node(qn).output_shapes(qn, [[300, 130]]) == [[300, 130], [3, 2]]
    qn["attrs"] = {}
    assert r.create_operator_for_node(qn).output_shapes(qn, [[4, 300, 130]]) == [[4, 300, 130], [4, 300, 2]]
    mn = {"op": "MatMulBlockScaled", "domain": "b200", "inputs": ["a", "as", "b", "bs"], "outputs": ["y"],
          "attrs": {"dtype": 16, "relu": 1}}
    mm = r.create_operator_for_node(mn)
    assert mm.dtype == torch.bfloat16 and mm.relu
    assert mm.output_shapes(mn, [[2, 5, 64], None, [100, 64], None]) == [[2, 5, 100]]
    with pytest.raises(ob.ValidationError):
        mm.validate({"inputs": ["a", "as", "b"], "outputs": ["y"]})
    with pytest.raises(ob.ValidationError):
        r.create_operator_for_node({**mn, "attrs": {"dtype": 7}})


def test_operators_are_copied_and_pickled_after_a_call(ob):
    """What a call keeps holds pointers to this process's descriptors: it stays out of copies."""
    import copy
    import pickle
    import types

    for op in (ob.RMSNormalization(1e-6, quantize=True), ob.QuantizeBlocks(128), ob.MatMulBlockScaled(torch.float16, True)):
        op._described(types.SimpleNamespace(device=0), lambda h, x: (ctypes.byref(C_INT),), torch.zeros(3))
        for other in (copy.copy(op), copy.deepcopy(op), pickle.loads(pickle.dumps(op))):
            assert type(other) is type(op) and other._settings() == op._settings()
            assert "_kept" in op.__dict__ and "_kept" not in other.__dict__


C_INT = ctypes.c_int()


def test_module_for_repeated_calls(ob, C):
    """Plans are checked when they are made, and fit nothing on the CPU."""
    calls = ob.ops._calls
    if calls is None:
        pytest.skip("onnx-rs_b200/_calls.so is not built")
    x, d = torch.zeros(2, 3), quant_desc(C)
    spec = ((2, 3), (3, 1), torch.float32)
    args = (1, 1, ctypes.addressof(d), d, 0)  # addresses that nothing calls
    plan = calls.Plan(*args, (x, None), (spec, spec), (0, -1, -2))
    assert calls.run([], 1, 0, 0, x, None) is None
    assert calls.run([plan], 1, 0, 0, x, None) is None  # a CPU tensor
    assert calls.run([plan], 1, 1, 0, x, None) is None  # another device's handle
    assert calls.run([plan], 0, 0, 0, x, None) is None  # no handle
    assert calls.run([plan, object()], 1, 0, 0, x) is None
    assert calls.run([plan], 1, 0, 0, x, 5) is None
    for ins, outs, slots in (((x,) * 6, (spec,), (0, -1, -1)), ((x,), (spec,), (0, -1)), ((x,), (spec,), (1, -1, -1)),
                             ((x,), (spec,), (0, -1, -2)), ((3,), (spec,), (0, -1, -1)), ((x,), (((2,), (1, 1), torch.float32),), (0, -1, -1)),
                             ((x,), (((2,), (1,), 5),), (0, -1, -1))):
        with pytest.raises(ValueError):
            calls.Plan(*args, ins, outs, slots)
    with pytest.raises(TypeError):
        calls.run()
    with pytest.raises(TypeError):
        calls.run((plan,), 1, 0, 0, x, None)
    with pytest.raises(TypeError):
        calls.Plan(*args, [x], (spec,), (0, -1, -1))


@pytest.mark.parametrize("rows,row,block", [(1 << 28, 1 << 36, 1 << 36), (1 << 30, 1 << 34, 1 << 34),
                                            (1 << 27, 1 << 37, 1 << 37)])
def test_scales_that_overlap_far_apart(C, rows, row, block):
    """Scales (i, j) and (i + 1, j - 1) in one place, with strides whose products pass 64 bits."""
    assert call_norm(C, norm_desc(C, rows=rows, out_type=E4M3, y_scale_row=row, y_scale_block=block)) == C.ERR_VALIDATION
    assert call_quant(C, quant_desc(C, rows=rows, scale_row=row, scale_block=block)) == C.ERR_VALIDATION


def test_scales_side_by_side_at_the_edge(C):
    """The closest strides that do not overlap are taken, both ways round."""
    for row, block in ((2, 1), (1, 4), (3, 1), (1, 5), (1 << 37, 1 << 36), (1 << 35, 1 << 37)):
        assert call_norm(C, norm_desc(C, out_type=E4M3, y_scale_row=row, y_scale_block=block)) == C.ERR_INVALID_ARGUMENT
        assert call_quant(C, quant_desc(C, scale_row=row, scale_block=block)) == C.ERR_INVALID_ARGUMENT


@pytest.fixture
def kept_op(ob, monkeypatch):
    """An operator that keeps its calls, with plans that only name the settings they were made under;
    on_plan is called while a plan is made."""
    import types

    class Op(ob.ops._Described, ob.ops.Operator):
        entry, slots, setting, on_plan = "onnxb200_quantize_blocks", (0, -1, -1), 0, None

        def _settings(self):
            return self.setting

        def _describe(self, h, x):
            return ob._capi.QuantizeDesc(rows=self.setting), (((2,), (1,), torch.float32),), ()

        def see(self, size):
            return self._described(types.SimpleNamespace(device=0), self._prepare, torch.zeros(size))

    op = Op()

    def plan(entry, get_stream, address, desc, device, tensors, outputs, slots):
        if Op.on_plan:
            Op.on_plan()
        return types.SimpleNamespace(setting=desc.rows, size=tensors[0].numel())

    monkeypatch.setattr(ob.ops, "_calls", types.SimpleNamespace(Plan=plan))
    return op


def test_settings_changed_while_a_call_is_described(kept_op):
    """As by another thread: the call goes through, and nothing made under the old settings is kept."""
    def change():
        type(kept_op).on_plan = None
        kept_op.setting = 5

    type(kept_op).on_plan = staticmethod(change)
    assert kept_op.see(3).plan.setting == 0
    assert not kept_op._plans
    assert kept_op.see(3).plan.setting == 5
    assert [p.setting for p in kept_op._plans] == [5]


def test_layouts_dropped_while_a_call_is_described(kept_op):
    """Another thread sees so many layouts in the meantime that the oldest are dropped."""
    def others():
        type(kept_op).on_plan = None
        for i in range(64):
            kept_op.see(100 + i)

    type(kept_op).on_plan = staticmethod(others)
    assert kept_op.see(3).plan.size == 3
    assert kept_op._plans[0].size == 3 and len(kept_op._plans) <= 64


def test_operator_shared_by_threads(kept_op):
    """Layouts and settings seen by several threads at once: no call fails, and every plan that is kept
    was made under the settings of now."""
    import sys
    import threading
    errors, stop = [], threading.Event()

    def see(seed):
        try:
            i = 0
            while not stop.is_set():
                i += 1
                got = kept_op.see(1 + (seed * 31 + i) % 97)
                plans = kept_op._plans
                assert got.plan is not None and (plans is None or len({p.setting for p in plans}) <= 1)
        except Exception as e:  # noqa: BLE001 -- handed to the test's thread
            errors.append(e)

    was = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    threads = [threading.Thread(target=see, args=(i,)) for i in range(4)]
    try:
        for t in threads:
            t.start()
        for i in range(300):
            kept_op.setting = i
    finally:
        stop.set()
        for t in threads:
            t.join()
        sys.setswitchinterval(was)
    assert not errors, errors[0]
    for i in range(3):
        kept_op.see(i)
    assert all(p.setting == 299 for p in kept_op._plans)


def test_the_oldest_layout_is_dropped(kept_op):
    """A call with a 65th layout takes the place of the first: the others stay as they were kept."""
    first = [kept_op.see(i) for i in range(64)]
    kept_op.see(64)
    assert len(kept_op._kept) == 64
    assert [p.size for p in kept_op._plans] == list(range(64, 0, -1))
    assert all(kept_op.see(i) is first[i] for i in range(1, 64))
    assert kept_op.see(0) is not first[0]


def test_norm_output_in_the_type_of_the_weight(ob, C):
    """ONNX gives y the scale's type: taken by the entry, and what operators made from nodes ask for."""
    assert call_norm(C, norm_desc(C, weight_type=F32, out_type=F32)) == C.ERR_INVALID_ARGUMENT
    assert call_norm(C, norm_desc(C, weight_type=F16, out_type=F16)) == C.ERR_INVALID_ARGUMENT
    assert call_norm(C, norm_desc(C, weight_type=F32, out_type=F16)) == C.ERR_VALIDATION
    assert call_norm(C, norm_desc(C, weight_type=F32, out_type=F32), y=ctypes.c_void_p(4098)) == C.ERR_VALIDATION
    node = {"op": "RMSNormalization", "inputs": ["x", "w"], "outputs": ["y"], "attrs": {}}
    r = ob.OperatorRegistry.initialize_standard_operators()
    assert r.create_operator_for_node(node, opset=23).y_like == "scale"
    assert ob.RMSNormalization().y_like == ob.RMSNormalization.from_node(node, y_like="x").y_like == "x"
    with pytest.raises(ob.ValidationError):
        ob.RMSNormalization(y_like="residual")


def test_norm_refuses_other_stash_types(ob):
    """Sums are fp32: a node that asks for another type of its intermediate values is not silently taken."""
    node = {"op": "RMSNormalization", "inputs": ["x", "w"], "outputs": ["y"], "attrs": {"stash_type": 1}}
    assert ob.RMSNormalization.from_node(node).epsilon == 1e-5
    for t in (10, 11, 16):
        node["attrs"]["stash_type"] = t
        with pytest.raises(ob.UnsupportedFeature):
            ob.RMSNormalization.from_node(node)


def test_quantize_shapes_are_refused_as_the_call_is(ob):
    """Weights are 2-D, activations have a last axis: shape inference says so before a call does."""
    node = {"op": "QuantizeBlocks", "inputs": ["x"], "outputs": ["q", "s"], "attrs": {"block_rows": 128}}
    op = ob.QuantizeBlocks(128)
    for shape in ([300], [4, 300, 130], []):
        with pytest.raises(ob.ValidationError):
            op.output_shapes(node, [shape])
    assert op.output_shapes(node, [None]) == [None, None]
    node["attrs"] = {}
    assert ob.QuantizeBlocks().output_shapes(node, [[300]]) == [[300], [3]]
    with pytest.raises(ob.ValidationError):
        ob.QuantizeBlocks().output_shapes(node, [[]])


def test_settings_changed_after_construction_are_checked(ob, monkeypatch):
    """As the constructor checks them, at the next call."""
    monkeypatch.setattr(ob.ops, "_check_device", lambda *a: None)
    x, w = torch.zeros(4, 256), torch.ones(256)
    norm = ob.RMSNormalization()
    norm._describe(None, x, w, None)
    norm.y_like = "weight"
    with pytest.raises(ob.ValidationError):
        norm._describe(None, x, w, None)
    e4m3 = torch.zeros(4, 256).to(torch.float8_e4m3fn)
    mm = ob.MatMulBlockScaled()
    mm._describe(None, e4m3, torch.ones(4, 2), e4m3, torch.ones(1, 2), None)
    mm.dtype = torch.float64
    with pytest.raises(ob.ValidationError):
        mm._describe(None, e4m3, torch.ones(4, 2), e4m3, torch.ones(1, 2), None)


def test_settings_changed_by_a_finaliser(ob, kept_op):
    """The collector may run one wherever a list grows, so also while what is kept is published."""
    import threading

    def finalise():
        with ob.ops._keeping:  # as a thread that publishes
            kept_op.setting = 7

    t = threading.Thread(target=finalise, daemon=True)
    t.start()
    t.join(10)
    assert not t.is_alive() and kept_op.see(3).plan.setting == 7
