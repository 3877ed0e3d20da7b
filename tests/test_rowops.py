"""CPU: what the row operators (per-row quantisation, products with epilogue,
products grouped by expert, log probabilities) refuse, through the C ABI and
through dlq_amd.ops -- no call here reaches the GPU."""
import ctypes as C

import pytest
import torch

P = 4096  # an address that passes for an aligned pointer; never read


def desc(**kw):
    from dlq_amd.lib import LinearDesc
    d = dict(M=4, N=8, K=32, ldx=32, ldw=32, ldy=8, ldr=8, act=0, out_type=1) | kw
    return LinearDesc(*[d[n] for n, _ in LinearDesc._fields_])


def linear(fn, d, x=P, xs=P, w=P, ws=P, bias=P, res=None, y=P, grouped=None):
    from dlq_amd.lib import lib
    f = getattr(lib, fn)
    head = (C.byref(d),) if grouped is None else (C.byref(d),) + grouped
    return f(*head, x, xs, w, ws, bias, res, y, None), lib.dlq_last_error().decode()


FNS = ["dlq_linear_act_s8", "dlq_linear_act_f8"]
GFNS = ["dlq_linear_grouped_s8", "dlq_linear_grouped_f8"]

BAD_DESC = [(dict(M=-1), "shape"), (dict(N=-1), "shape"), (dict(K=-1), "shape"),
            (dict(K=131072, ldx=131072, ldw=131072), "131071"), (dict(act=5), "act"), (dict(act=-1), "act"),
            (dict(out_type=2), "out_type"), (dict(ldx=31), "below K"), (dict(ldw=31), "below K"),
            (dict(ldy=7), "below N")]


@pytest.mark.parametrize("fn", FNS + GFNS)
@pytest.mark.parametrize("bad,word", BAD_DESC, ids=[str(b) for b, _ in BAD_DESC])
def test_linear_refuses_bad_desc(fn, bad, word):
    rc, msg = linear(fn, desc(**bad), grouped=(2, P) if fn in GFNS else None)
    assert rc == 1 and word in msg, (rc, msg)


@pytest.mark.parametrize("fn", FNS + GFNS)
@pytest.mark.parametrize("size", [2 ** 31 - 511, 2 ** 31 - 1])
def test_linear_refuses_sizes_next_to_2_31(fn, size):
    """Row and column numbers of the last tile would not be an int's."""
    for kw in (dict(M=size), dict(N=size, ldy=size)):
        rc, msg = linear(fn, desc(**kw), x=None, grouped=(2, P) if fn in GFNS else None)
        assert rc == 1 and "2^31 - 512" in msg, (rc, msg)


@pytest.mark.parametrize("fn", FNS + GFNS)
def test_linear_refuses_pointers(fn):
    g = (2, P) if fn in GFNS else None
    for kw in (dict(x=None), dict(w=None), dict(ws=None), dict(y=None)):
        rc, msg = linear(fn, desc(), grouped=g, **kw)
        assert rc == 1 and "null" in msg, (kw, rc, msg)
    for kw in (dict(xs=P + 2), dict(ws=P + 1), dict(bias=P + 3), dict(y=P + 1), dict(res=P + 1)):
        rc, msg = linear(fn, desc(), grouped=g, **kw)
        assert rc == 1 and "aligned" in msg, (kw, rc, msg)
    rc, msg = linear(fn, desc(ldr=7), res=P, grouped=g)
    assert rc == 1 and "below N" in msg
    rc, msg = linear(fn, desc(ldr=16), res=P, grouped=g)
    assert rc == 1 and "another row stride" in msg
    # nothing to do is no error, and touches nothing
    assert linear(fn, desc(M=0), x=None, w=None, ws=None, y=None, grouped=g)[0] == 0
    assert linear(fn, desc(N=0, ldy=0), x=None, w=None, ws=None, y=None, grouped=g)[0] == 0


@pytest.mark.parametrize("fn", FNS + GFNS)
def test_fp8_sums_belong_to_e4m3(fn):
    """The flag beside an activation: unknown to int8, no activation by itself."""
    g = (2, P) if fn in GFNS else None
    for act in (256, 256 + 4):
        rc, msg = linear(fn, desc(act=act, M=0), grouped=g)
        assert (rc == 1 and "bad act" in msg) if fn.endswith("s8") else rc == 0
    for act in (256 + 5, 512, 512 + 256, -256):
        rc, msg = linear(fn, desc(act=act, M=0), grouped=g)
        assert rc == 1 and "bad act" in msg


@pytest.mark.parametrize("fn", FNS + GFNS)
def test_linear_refuses_more_tiles_than_a_launch_takes(fn):
    g = (2, P) if fn in GFNS else None
    n = 2 ** 31 - 512
    for kw in (dict(M=n, N=n, ldy=n), dict(M=1, N=n, ldy=n), dict(M=1 << 20, N=n, K=33, ldx=33, ldw=33, ldy=n)):
        rc, msg = linear(fn, desc(**kw), grouped=g)
        assert rc == 1 and "more tiles" in msg, (kw, rc, msg)


@pytest.mark.parametrize("fn", GFNS)
def test_grouped_refuses(fn):
    rc, msg = linear(fn, desc(), grouped=(2, None))
    assert rc == 1 and "offsets" in msg
    assert linear(fn, desc(), grouped=(-1, P))[0] == 1
    assert linear(fn, desc(), grouped=(65536, P))[0] == 1
    assert linear(fn, desc(), grouped=(2, P + 2))[0] == 1
    assert linear(fn, desc(), grouped=(0, P))[0] == 0  # no experts: no rows


@pytest.mark.parametrize("fn", ["dlq_quantize_rows_dyn_s8", "dlq_quantize_rows_dyn_f8"])
def test_quantize_rows_dyn_refuses(fn):
    from dlq_amd.lib import lib
    f = getattr(lib, fn)

    def call(x=P, t=0, rows=3, cols=8, ldx=8, q=P, ldq=8, scale=P):
        return f(x, t, rows, cols, ldx, q, ldq, scale, None)

    for kw in (dict(rows=-1), dict(cols=0), dict(t=2), dict(t=-1), dict(ldx=7), dict(ldq=7), dict(x=None),
               dict(q=None), dict(scale=None), dict(x=P + 2), dict(x=P + 1, t=1), dict(scale=P + 1)):
        assert call(**kw) == 1, kw
    assert call(rows=0, x=None, q=None, scale=None) == 0


def test_logprobs_refuses():
    from dlq_amd.lib import lib

    def call(x=P, t=0, rows=3, K=100, ldx=100, tokens=P, top=4, lp=P, ent=P, ti=P, tl=P, ws=P, nb=1 << 40):
        return lib.dlq_logprobs(x, t, rows, K, ldx, tokens, top, lp, ent, ti, tl, ws, nb, None)

    for kw in (dict(rows=-1), dict(K=0, ldx=0, top=0), dict(t=2), dict(ldx=99), dict(top=-1), dict(top=65),
               dict(K=3, top=4), dict(x=None), dict(tokens=None), dict(lp=None), dict(ti=None), dict(tl=None),
               dict(x=P + 2), dict(tokens=P + 2), dict(ent=P + 2), dict(ti=P + 1), dict(tl=P + 1)):
        assert call(**kw) == 1, kw
    assert call(rows=0, x=None) == 0
    need = lib.dlq_logprobs_workspace_bytes(3, 1 << 20, 4)
    if need:
        assert call(K=1 << 20, ldx=1 << 20, nb=need - 1) == 1
        assert call(K=1 << 20, ldx=1 << 20, ws=None) == 1
        assert call(K=1 << 20, ldx=1 << 20, ws=P + 4) == 1


def test_ops_refuse_host_tensors():
    from dlq_amd import ops
    x, w, s = torch.zeros(4, 32, dtype=torch.int8), torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8)
    with pytest.raises(TypeError):
        ops.linear_act_s8(x, w, None, s)
    with pytest.raises(TypeError):
        ops.linear_act_f8(x, w, None, s)
    with pytest.raises(ValueError):
        ops.linear_act_s8(x, w, None, s, act="tanh")
    with pytest.raises(TypeError):
        ops.linear_act_s8(x, w, None, s, out_dtype=torch.float16)
    with pytest.raises(TypeError):
        ops.linear_grouped_s8(x, None, w[None], None, s[None])
    with pytest.raises(TypeError):
        ops.quantize_rows_dyn_s8(torch.zeros(2, 8))
    with pytest.raises(TypeError):
        ops.logprobs(torch.zeros(2, 8))


class Placed(torch.Tensor):
    """Passes for a tensor on device 0; without memory."""
    is_cuda = True

    def get_device(self):
        return 0


def placed(dtype, rows, cols, ld=None):
    ld = cols if ld is None else ld
    big = torch.empty(max(rows - 1, 0) * ld + cols, dtype=dtype, device="meta")
    return big.as_strided((rows, cols), (ld, 1)).as_subclass(Placed)


@pytest.mark.parametrize("ld", [2 ** 31, 2 ** 32 + 32, 2 ** 32 + 2 ** 31])
def test_ops_refuse_strides_past_32_bits(ld):
    """A row stride that an int does not hold is refused, not cut to its low bits."""
    from dlq_amd import ops
    x, w, s = placed(torch.int8, 4, 32), placed(torch.int8, 8, 32), placed(torch.float32, 1, 8)[0]
    far = lambda t, c: placed(t, 4, c, ld)  # noqa: E731
    e = placed(torch.int32, 1, 2)[0]
    word = "strides end at 2147483647"
    for f in (ops.linear_act_s8, ops.linear_act_f8):
        code = torch.int8 if f is ops.linear_act_s8 else torch.uint8
        y, v = placed(code, 4, 32), placed(code, 8, 32)
        with pytest.raises(ValueError, match="x: .*" + word):
            f(far(code, 32), v, None, s)
        with pytest.raises(ValueError, match="w: .*" + word):
            f(y, far(code, 32), None, s[:4])
        with pytest.raises(ValueError, match="out: .*" + word):
            f(y, v, None, s, out=far(torch.float32, 8))
        with pytest.raises(ValueError, match="residual: .*" + word):
            f(y, v, None, s, residual=far(torch.float32, 8))
    with pytest.raises(ValueError, match="x: .*" + word):
        ops.linear_grouped_s8(far(torch.int8, 32), e, w[None], None, s[None])
    with pytest.raises(ValueError, match="out: .*" + word):
        ops.linear_grouped_s8(x, e, w[None], None, s[None], out=far(torch.float32, 8))
    for f in (ops.quantize_rows_dyn_s8, ops.quantize_rows_dyn_f8):
        with pytest.raises(ValueError, match="x: .*" + word):
            f(far(torch.bfloat16, 32))
        with pytest.raises(ValueError, match="ld: "):
            f(placed(torch.bfloat16, 4, 32), ld=ld)
    with pytest.raises(ValueError, match="x: .*" + word):
        ops.logprobs(far(torch.float32, 32))


def test_ops_refuse_sizes_past_32_bits():
    from dlq_amd import ops
    n = 2 ** 32 + 1
    s = placed(torch.float32, 1, 8)[0]
    for x in (placed(torch.int8, n, 1), placed(torch.int8, 1, n)):
        with pytest.raises(ValueError, match="sizes"):
            ops.linear_act_s8(x, placed(torch.int8, 8, x.shape[1]), None, s)
    with pytest.raises(ValueError, match="sizes"):
        ops.linear_act_s8(placed(torch.int8, 4, 1), placed(torch.int8, n, 1), None, placed(torch.float32, 1, n)[0])
    with pytest.raises(ValueError, match="sizes"):
        ops.linear_grouped_s8(placed(torch.int8, 4, 1), placed(torch.int32, 1, 2)[0], placed(torch.int8, n, 1)[None],
                              None, placed(torch.float32, 1, n))
    with pytest.raises(ValueError, match="sizes"):
        ops.quantize_rows_dyn_s8(placed(torch.float32, n, 1))
    with pytest.raises(ValueError, match="ld: "):
        ops.quantize_rows_dyn_s8(placed(torch.float32, 4, 32), ld=31)
    with pytest.raises(ValueError, match="sizes"):
        ops.logprobs(placed(torch.float32, n, 1))
    for top in (-1, 65, 2 ** 32 + 3):
        with pytest.raises(ValueError, match="top"):
            ops.logprobs(placed(torch.float32, 4, 100), None, top)
