"""The operators on 8-bit rows against 64-bit arithmetic: whole numbers exactly, everything else within the roundings of float32 that stand
between (2^-24 each) and one rounding to the output's type."""
import math

import pytest
import torch

from test_gpu_kernels import DEV, _ops

pytestmark = pytest.mark.gpu

F32, BF = torch.float32, torch.bfloat16
U = 2.0 ** -24                                     # half a step of float32, relative


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _codes(x):
    """(q, s) of float64 rows by the definition; torch.round takes ties to even.  127 x / top: 127 x is exact in 64 bits, and a quotient that is
    not half way between two whole numbers is further from there than its rounding (numerators below 2^31, denominators below 2^24)."""
    top = x.abs().amax(1, keepdim=True)
    q = torch.nan_to_num(torch.round(127 * x / top), 0.0, 0.0, 0.0)
    bad = ~torch.isfinite(x).all(1)
    q[bad] = 0
    s = (top / 127)[:, 0]
    s[bad] = math.nan
    return q.to(torch.int8), s


def _fresh(rows, width, fill=77):
    """Room for rows with one row behind them, all bytes `fill`; (q, the whole buffer)."""
    whole = torch.full((rows + 1, -(-width // 16) * 16), fill, dtype=torch.int8, device=DEV)
    return whole[:rows, :width], whole


def _untouched(whole, rows, width, fill=77):
    return bool((whole[:rows, width:] == fill).all()) and bool((whole[rows:] == fill).all())


def _same_scale(s, want, ulps=2.0):
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(s), nan)
    # (a scale below 2^-126 is a whole number of 2^-149)
    assert ((s.double() - want)[~nan].abs() <= 2 * ulps * U * want[~nan].abs() + 2.0 ** -149).all()


def _x(rows, width, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + rows * 7 + width)
    x = torch.randn(rows, width, generator=g, device=DEV)
    return (x * torch.exp(2 * torch.randn(rows, 1, generator=g, device=DEV))).to(dtype)


WIDTHS = [1, 2, 7, 8, 15, 16, 17, 31, 33, 64, 127, 129, 255, 256, 512, 1000, 1024, 1531, 2048, 2056, 4096, 4100, 6144, 8192, 8200, 14336, 16384, 16400, 28672,
          28673, 32768, 40001, 70000]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("width", WIDTHS)
def test_rows_become_integers_and_are_read_back(width, dtype):
    ops = _ops()
    for rows in (1, 3, 41):
        x = _x(rows, width, dtype)
        q, whole = _fresh(rows, width)
        s = torch.full((rows + 1,), 5.0, device=DEV)
        ops.quantize_q8(q, s[:rows], x)
        want_q, want_s = _codes(x.double())
        assert torch.equal(q, want_q)
        _same_scale(s[:rows], want_s)
        assert _untouched(whole, rows, width) and s[rows] == 5.0
        for out_dtype in (F32, BF):
            y = torch.full((rows + 1, width), 3.0, dtype=out_dtype, device=DEV)
            ops.dequantize_q8(y[:rows], q, s[:rows])
            assert torch.equal(y[:rows], (q.float() * s[:rows, None]).to(out_dtype)) and (y[rows] == 3.0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("width", [16, 40, 1024, 1531, 4096, 9000])
def test_many_rows(width, dtype):
    """More rows than blocks that are on the device at one time, as wide as narrow."""
    ops = _ops()
    rows = 5000
    x = _x(rows, width, dtype)
    q, whole = _fresh(rows, width)
    s = torch.empty(rows, device=DEV)
    ops.quantize_q8(q, s, x)
    want_q, want_s = _codes(x.double())
    assert torch.equal(q, want_q) and _untouched(whole, rows, width)
    _same_scale(s, want_s)
    y = torch.empty(rows, width, dtype=dtype, device=DEV)
    ops.dequantize_q8(y, q, s)
    assert torch.equal(y, (q.float() * s[:, None]).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_rows_of_wider_buffers_and_odd_addresses(dtype):
    ops = _ops()
    for rows, width, offset, step in ((9, 300, 1, 333), (9, 4096, 3, 4104), (5, 1024, 8, 2048), (4, 57, 0, 64), (3, 14336, 4, 14344)):
        x = torch.empty(rows * step + offset, dtype=dtype, device=DEV)[offset:].view(rows, step)[:, :width]
        x.copy_(_x(rows, width, dtype))
        whole = torch.full((rows, 2 * (-(-width // 16) * 16)), 77, dtype=torch.int8, device=DEV)
        at = 0 if width % 32 else -(-width // 16) * 16
        q = whole[:, at:at + width]
        s = torch.empty(rows, device=DEV)
        ops.quantize_q8(q, s, x)
        want_q, want_s = _codes(x.double())
        assert torch.equal(q, want_q)
        _same_scale(s, want_s)
        q.fill_(77)
        assert (whole == 77).all()
        q.copy_(want_q)
        back = torch.full((rows * step + offset,), 3.0, dtype=dtype, device=DEV)
        y = back[offset:].view(rows, step)
        ops.dequantize_q8(y[:, :width], q, s)
        assert torch.equal(y[:, :width], (q.float() * s[:, None]).to(dtype)) and (y[:, width:] == 3.0).all() and (back[:offset] == 3.0).all()
        total = torch.full((rows * step + offset,), 3.0, dtype=dtype, device=DEV)[offset:].view(rows, step)
        gain = torch.ones(width + 1, dtype=dtype, device=DEV)[1:]
        add = torch.zeros(rows * step + offset, dtype=BF, device=DEV)[offset:].view(rows, step)[:, :width]
        q.fill_(0)
        ops.rmsnorm_q8(q, s, x, gain, 1e-5, add=add, total=total[:, :width])
        assert torch.equal(q, want_q) and torch.equal(total[:, :width], x) and (total[:, width:] == 3.0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("width", [1, 3, 8, 17, 41, 255, 263, 777, 1023, 1033, 4111, 9001, 17001, 33001])
def test_rows_that_begin_anywhere(width, dtype):
    """Every place of a row's begin within 16 bytes (rows of odd length have them all), what lies around the rows untouched, the sums in place."""
    ops = _ops()
    rows = 11
    for offset, step in ((0, width), (1, width + 1), (2, width + 2), (3, width), (5, width + 7)):
        def buffer(kind, fill):
            flat = torch.full((rows * step + offset + 8,), fill, dtype=kind, device=DEV)
            return flat, flat[offset:offset + rows * step].view(rows, step)[:, :width]

        def around(flat, fill):
            mask = torch.ones(flat.numel(), dtype=torch.bool, device=DEV)
            mask[offset:offset + rows * step].view(rows, step)[:, :width] = False
            return bool((flat[mask] == fill).all())
        flat_x, x = buffer(dtype, 5.0)
        x.copy_(_x(rows, width, dtype, offset))
        q, whole = _fresh(rows, width)
        s = torch.empty(rows, device=DEV)
        ops.quantize_q8(q, s, x)
        want_q, want_s = _codes(x.double())
        assert torch.equal(q, want_q) and _untouched(whole, rows, width)
        _same_scale(s, want_s)
        flat_y, y = buffer(dtype, 3.0)
        ops.dequantize_q8(y, q, s)
        assert torch.equal(y, (q.float() * s[:, None]).to(dtype)) and around(flat_y, 3.0)
        flat_a, a = buffer(BF if offset % 2 else F32, 9.0)
        a.copy_(_x(rows, width, a.dtype, 40 + offset))
        gain = (1 + 0.2 * torch.randn(width + offset, device=DEV)).to(dtype)[offset:]
        t = (x.float() + a.float()).to(dtype)
        want_q = _codes((t.float() * gain.float()).double())[0]
        flat_t, total = buffer(dtype, 4.0)
        s2 = torch.empty(rows, device=DEV)
        ops.rmsnorm_q8(q, s, x, gain, 1e-5, add=a, total=total)
        assert torch.equal(q, want_q) and torch.equal(total, t) and around(flat_t, 4.0)
        ops.rmsnorm_q8(q, s2, x, gain, 1e-5, add=a, total=x)
        assert torch.equal(q, want_q) and torch.equal(x, t) and around(flat_x, 5.0) and torch.equal(s, s2)
        # the sums are added in the same order wherever a row begins
        ops.rmsnorm_q8(q, s2, t.contiguous(), gain.clone(), 1e-5)
        assert torch.equal(q, want_q) and torch.equal(s, s2)


@pytest.mark.parametrize("width", [5, 64, 1024, 4096])
def test_borders_between_whole_numbers(width):
    """Entries exactly half way between two whole numbers go to the even one, their neighbours in float32 to their own side."""
    ops = _ops()
    for top in (127.0, 127.0 * 2 ** -20, 1.0, 3.0, 0.7265625, 1.9921875, 251.0):
        halves = (torch.arange(-127, 127, device=DEV) + 0.5).double() * top / 127
        exact = halves.float()
        near = torch.cat([exact, torch.nextafter(exact, torch.full_like(exact, 1e9)), torch.nextafter(exact, torch.full_like(exact, -1e9))])
        rows = -(-near.numel() // max(1, width - 1))
        x = torch.zeros(rows, width, device=DEV)
        x[:, 1:] = torch.nn.functional.pad(near, (0, rows * (width - 1) - near.numel())).view(rows, width - 1)
        x[:, 0] = torch.tensor(top, device=DEV)
        x[1::2, 0] *= -1
        for dtype in (F32, BF):
            xs = x.to(dtype)
            q, s = ops.q8_rows(rows, width, DEV), torch.empty(rows, device=DEV)
            ops.quantize_q8(q, s, xs)
            assert torch.equal(q, _codes(xs.double())[0])
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5, 125.5]], device=DEV)
    q, s = ops.q8_rows(1, 10, DEV), torch.empty(1, device=DEV)
    ops.quantize_q8(q, s, x)
    assert q.tolist() == [[127, 0, 2, 2, 0, -2, -2, 126, -126, 126]] and s.item() == 1.0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("width", [3, 100, 2048])
def test_the_ends_of_the_range(width, dtype):
    ops = _ops()
    base = _x(8, width, dtype, 3).double()
    base /= base.abs().amax(1, keepdim=True)
    x = torch.stack([base[0] * 2.0 ** -149 * 100, base[1] * 2.0 ** -130, base[2] * 2.0 ** -100, base[3] * 2.0 ** -61, base[4] * 2.0 ** 99,
                     base[5] * 2.0 ** 101, base[6] * 2.0 ** 127, base[7] * 0]).to(dtype)
    more = _x(5, width, dtype, 5)
    more[0, width - 1], more[1, 0], more[2, width // 2] = math.nan, math.inf, -math.inf
    more[3] = 0
    more[3, width - 1] = -0.0
    x = torch.cat([x, more])
    q, s = ops.q8_rows(13, width, DEV), torch.empty(13, device=DEV)
    ops.quantize_q8(q, s, x)
    want_q, want_s = _codes(x.double())
    assert torch.equal(q, want_q)
    _same_scale(s, want_s)
    assert torch.isnan(s[8:11]).all() and not torch.isnan(s[11:]).any() and s[7] == 0 and s[11] == 0
    values = torch.empty(13, width, device=DEV)
    ops.dequantize_q8(values, q, s)
    assert torch.isnan(values[8:11]).all() and (values[11] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("width", [1, 7, 16, 100, 512, 1024, 1531, 2048, 4096, 4104, 8192, 14336, 16384, 20000, 33000])
def test_norm_with_the_addition_in_front(width, dtype):
    ops = _ops()
    for rows, add_dtype, gain_dtype, in_place in ((1, BF, BF, True), (37, None, BF, False), (37, F32, F32, False), (6, BF, F32, False), (1300, BF, BF, True)):
        if rows * width > 1 << 24:
            continue
        x = _x(rows, width, dtype)
        gain = (1 + 0.2 * torch.randn(width, device=DEV)).to(gain_dtype)
        add = None if add_dtype is None else _x(rows, width, add_dtype, 9)
        t = x if add is None else (x.float() + add.float()).to(dtype)
        want_q, want_s = _codes((t.float() * gain.float()).double())
        eps = 1e-3
        want_s = want_s / torch.sqrt(t.double().pow(2).mean(1) + eps)
        q, whole = _fresh(rows, width)
        s = torch.empty(rows, device=DEV)
        # without a place for the sums, then with one
        ops.rmsnorm_q8(q, s, x, gain, eps, add=add)
        first = (q.clone(), s.clone())
        total = None if add is None else (x if in_place else torch.empty_like(x))
        ops.rmsnorm_q8(q, s, x, gain, eps, add=add, total=total)
        assert torch.equal(q, first[0]) and torch.equal(s, first[1]) and torch.equal(q, want_q) and _untouched(whole, rows, width)
        # the mean of the squares: a chain of width / 32 additions at most and a tree; half of that in the root, and five roundings more
        _same_scale(s, want_s, (width / 32 + 12) / 4 + 3)
        if add is not None:
            assert torch.equal(total, t)


def test_norm_of_rows_without_numbers():
    ops = _ops()
    x = _x(6, 300, F32)
    x[1, 7], x[2, 0], x[3] = math.nan, math.inf, 0
    add = torch.zeros(6, 300, dtype=BF, device=DEV)
    add[4, 299] = -math.inf
    gain = torch.ones(300, device=DEV)
    q, s = ops.q8_rows(6, 300, DEV), torch.empty(6, device=DEV)
    total = torch.empty_like(x)
    ops.rmsnorm_q8(q, s, x, gain, 0.0, add=add, total=total)
    assert torch.isnan(s[[1, 2, 3, 4]]).all() and (q[1:5] == 0).all() and torch.isfinite(s[[0, 5]]).all()       # (0 / 0 with eps 0: no number either)
    ops.rmsnorm_q8(q, s, x, gain, 1e-5)
    assert s[3] == 0 and torch.isfinite(s[[0, 3, 4, 5]]).all() and torch.isnan(s[[1, 2]]).all()
    assert torch.equal(torch.isnan(total), torch.isnan(x + add.float()))


# -- products -------------------------------------------------------------------------------------------------------------------
def _operands(T, rows_w, K, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + T * 3 + rows_w * 5 + K)
    a, w = _fresh(T, K, 111)[0], _fresh(rows_w, K, 111)[0]       # (what lies between the rows is not zero)
    for m in (a, w):
        m.copy_(torch.randint(-128, 128, m.shape, generator=g, device=DEV, dtype=torch.int8))
    sa = torch.exp(torch.randn(T, generator=g, device=DEV)) * 0.02
    sw = torch.exp(torch.randn(rows_w, generator=g, device=DEV)) / (3000 * math.sqrt(K))
    return a, sa, w, sw


def _silu(g):
    return g / (1 + torch.exp(-g))


def _check_product(T, N, K, epilogue, dtype, rule="silu", bias=False, seed=0):
    ops = _ops()
    gated = epilogue == ops.EPILOGUE_SWIGLU
    a, sa, w, sw = _operands(T, 2 * N if gated else N, K, seed)
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    base = torch.randn(T + 1, N, device=DEV).to(dtype)
    out = base.clone()
    glu = None if rule == "silu" else ops.GluRule("clamped", 1.5, 1.702)
    b = torch.randn(2 * N, device=DEV) if bias else None
    ops.gemm_q8_tc(out[:T], a, sa, w, sw, epilogue, status, glu=glu, glu_bias=b)
    y = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()          # whole numbers below 2^53: exact but for the scales
    err = 3 * U * y.abs()                                                        # the sum to float32, two products
    if epilogue == ops.EPILOGUE_ACCUMULATE:
        want = base[:T].double() + y
    elif gated:
        if bias:
            y = y + b.double()
            err = err + U * (y.abs() + err)
        g, u, eg, eu = y[:, :N], y[:, N:], err[:, :N], err[:, N:]
        if rule == "silu":
            h = _silu(g)
            want = h * u
            err = 1.1 * eg * (u.abs() + eu) + h.abs() * eu                       # |silu'| <= 1.1
        else:
            g, u = g.clamp(max=1.5), u.clamp(-1.5, 1.5)
            h = g * torch.sigmoid(1.702 * g)
            want = h * (u + 1)
            err = 1.1 * eg * ((u + 1).abs() + eu + U) + h.abs() * (eu + U * (u + 1).abs())
        # the exponential (2^-21 of itself, and its argument's rounding times the argument, which below -88 leaves nothing), the division, the products
        err = err + (2.0 ** -21 + 8 * U + 2 * U * (1.702 * g).abs().clamp(max=88)) * want.abs()
    else:
        want = y
    bound = err + _half_step(dtype) * (want.abs() + err) + 1e-37
    worst = ((out[:T].double() - want).abs() / bound).max().item()
    assert worst <= 1, (T, N, K, epilogue, dtype, worst)
    assert torch.equal(out[T], base[T])                                          # the row behind the last
    assert status.tolist() == [0, 0, 0, 0]
    return a, sa, w, sw, base, out, status


FORMS = [(0, F32), (0, BF), (1, F32), (2, F32), (2, BF)]


@pytest.mark.parametrize("T", [1, 2, 7, 16, 17, 31, 33, 64, 65, 97, 128, 129, 200, 256, 257, 300, 385, 512, 513, 700])
@pytest.mark.parametrize("N, K", [(1, 1), (8, 16), (100, 129), (128, 128), (130, 300), (257, 1000), (1024, 512)])
def test_products_in_every_form(T, N, K):
    for epilogue, dtype in FORMS:
        _check_product(T, N, K, epilogue, dtype)


@pytest.mark.parametrize("T", [1, 8, 40, 64, 100, 160, 300, 1000])
@pytest.mark.parametrize("N, K", [(2048, 2048), (2048, 6144), (512, 14336), (6144, 2048), (4096, 4096), (11000, 700), (333, 8191)])
def test_products_of_layers(T, N, K):
    for epilogue, dtype in FORMS:
        _check_product(T, N, K, epilogue, dtype)


@pytest.mark.parametrize("T, N, K", [(1, 1021, 1111), (33, 640, 512), (250, 256, 96), (531, 1021, 1111), (2000, 264, 200)])
def test_other_gates(T, N, K):
    for dtype in (F32, BF):
        for rule in ("silu", "clamped"):
            for bias in (False, True):
                if rule == "clamped" or bias:
                    _check_product(T, N, K, 2, dtype, rule, bias)


@pytest.mark.parametrize("T, N, K", [(3000, 4096, 2048), (4097, 1030, 999), (2048, 6144, 4096), (1777, 12288, 1024)])
def test_large_products(T, N, K):
    for epilogue, dtype in ((0, BF), (1, F32), (2, BF), (0, F32)):
        _check_product(T, N // 2 if epilogue == 2 else N, K, epilogue, dtype)


@pytest.mark.parametrize("T", [1, 70, 300])
def test_the_longest_rows(T):
    """All entries -128: the sums reach 128 * 128 * 131,071, the largest that 32 bits hold."""
    ops = _ops()
    K, N = ops.Q8_MAX_INNER, 140
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    a, w = ops.q8_rows(T, K, DEV), ops.q8_rows(N, K, DEV)
    a.fill_(-128); w.fill_(-128)
    w[1].fill_(127)
    ones = torch.ones(T, device=DEV), torch.ones(N, device=DEV)
    out = torch.empty(T, N, device=DEV)
    ops.gemm_q8_tc(out, a, ones[0], w, ones[1], ops.EPILOGUE_STORE, status)
    want = torch.full((T, N), float(128 * 128 * K), device=DEV)
    want[:, 1] = float(-128 * 127 * K)
    assert torch.equal(out, want) and status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("N, K, epilogue, dtype", [(2048, 2048, 0, BF), (2048, 6144, 1, F32), (1536, 1024, 2, BF), (4096, 4096, 0, F32), (100, 300, 2, F32)])
def test_a_row_does_not_depend_on_the_others(N, K, epilogue, dtype):
    ops = _ops()
    a, sa, w, sw, base, whole, status = _check_product(700, N, K, epilogue, dtype)
    for first, m in ((0, 1), (699, 1), (5, 16), (600, 33), (0, 64), (300, 128), (1, 129), (100, 257), (188, 512)):
        out = base[first:first + m].clone()
        ops.gemm_q8_tc(out, a[first:first + m], sa[first:first + m], w, sw, epilogue, status)
        assert torch.equal(out, whole[first:first + m]), m


@pytest.mark.parametrize("T", [5, 100, 300])
def test_outputs_inside_wider_buffers(T):
    """Rows further apart than they are long, at odd distances and addresses; operands that are pieces of wider rows."""
    ops = _ops()
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    for N, step, offset in ((100, 133, 1), (256, 512, 8), (130, 136, 0), (64, 64, 3)):
        for epilogue, dtype in FORMS:
            rows_w = 2 * N if epilogue == 2 else N
            a, sa, w, sw = _operands(T, rows_w, 512)
            plain = torch.zeros(T, N, dtype=dtype, device=DEV)
            ops.gemm_q8_tc(plain, a, sa, w, sw, epilogue, status)
            buffer = torch.full((T * step + offset,), 2.0, dtype=dtype, device=DEV)
            view = buffer[offset:].view(T, step)
            view[:, :N] = 0
            ops.gemm_q8_tc(view[:, :N], a, sa, w, sw, epilogue, status)
            assert torch.equal(view[:, :N], plain) and (view[:, N:] == 2.0).all() and (buffer[:offset] == 2.0).all()
            # the inner pieces of the rows
            part = torch.zeros(T, N, dtype=dtype, device=DEV)
            ops.gemm_q8_tc(part, a[:, 128:400], sa, w[:, 128:400], sw, ops.EPILOGUE_SWIGLU if epilogue == 2 else ops.EPILOGUE_STORE, status)
            again = torch.zeros(T, N, dtype=dtype, device=DEV)
            ops.gemm_q8_tc(again, a[:, 128:400].clone(), sa, w[:, 128:400].clone(), sw, ops.EPILOGUE_SWIGLU if epilogue == 2 else ops.EPILOGUE_STORE, status)
            assert torch.equal(part, again)
    assert status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("T", [4, 200])
def test_tokens_without_numbers_stay_without(T):
    ops = _ops()
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    x = torch.randn(T, 256, device=DEV)
    x[1, 3], x[3, 0] = math.nan, math.inf
    a, sa = ops.q8_rows(T, 256, DEV), torch.empty(T, device=DEV)
    ops.quantize_q8(a, sa, x)
    _, _, w, sw = _operands(T, 256, 256)
    for rule in (None, ops.GluRule("clamped", 1.5, 1.702)):
        out = torch.empty(T, 128, device=DEV)
        ops.gemm_q8_tc(out, a, sa, w, sw, ops.EPILOGUE_SWIGLU, status, glu=rule)
        bad = torch.isnan(out).all(1)
        assert bad.nonzero().flatten().tolist() == [1, 3] and torch.isfinite(out[~bad]).all()


def test_no_rows():
    ops = _ops()
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    a, sa, w, sw = _operands(4, 32, 64)
    ops.gemm_q8_tc(torch.empty(0, 32, device=DEV), a[:0], sa[:0], w, sw, ops.EPILOGUE_STORE, status)
    ops.gemm_q8_tc(torch.empty(4, 0, device=DEV), a, sa, w[:0], sw[:0], ops.EPILOGUE_STORE, status)
    ops.quantize_q8(a[:0], sa[:0], torch.empty(0, 64, device=DEV))
    ops.dequantize_q8(torch.empty(0, 64, device=DEV), a[:0], sa[:0])
    ops.rmsnorm_q8(a[:0], sa[:0], torch.empty(0, 64, device=DEV), torch.empty(64, device=DEV), 1e-5)
    torch.cuda.synchronize()


def _feed_forward(st, x, add, out, act, status):
    """norm, gate and up, 8-bit rows, down: as a layer runs them."""
    ops = _ops()
    T, hidden = x.shape
    q, s = ops.q8_rows(T, hidden, DEV), torch.empty(T, device=DEV)
    ops.rmsnorm_q8(q, s, x, st["gain"], 1e-5, add=add, total=x)
    ops.gemm_q8_tc(act, q, s, *st["w_in"], ops.EPILOGUE_SWIGLU, status)
    qa, sa = ops.q8_rows(T, act.shape[1], DEV), torch.empty(T, device=DEV)
    ops.quantize_q8(qa, sa, act)
    ops.gemm_q8_tc(out, qa, sa, *st["w_down"], ops.EPILOGUE_STORE, status)
    return qa, sa


@pytest.mark.parametrize("T", [1, 8, 77, 300])
def test_a_feed_forward_as_a_layer_runs_it(T):
    """Each step against 64 bits from what the step before left; then eagerly on another stream, and captured and replayed, with the same bits."""
    ops = _ops()
    hidden, inner = 512, 1100
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    st = {"gain": (1 + 0.1 * torch.randn(hidden, device=DEV)).bfloat16()}
    for name, rows, width in (("w_in", 2 * inner, hidden), ("w_down", hidden, inner)):
        w = torch.randn(rows, width, device=DEV) / math.sqrt(width)
        st[name] = (ops.q8_rows(rows, width, DEV), torch.empty(rows, device=DEV))
        ops.quantize_q8(*st[name], w)
    x0, add = torch.randn(T, hidden, device=DEV) * 3, torch.randn(T, hidden, device=DEV).bfloat16()
    x, act, out = x0.clone(), torch.empty(T, inner, dtype=BF, device=DEV), torch.empty(T, hidden, dtype=BF, device=DEV)
    qa, sa = _feed_forward(st, x, add, out, act, status)
    t = (x0.double() + add.double()).float()
    assert torch.equal(x, t)
    q, s = _codes((t * st["gain"].float()).double())
    s = s / torch.sqrt(t.double().pow(2).mean(1) + 1e-5)
    y = (q.double() @ st["w_in"][0].double().T) * s[:, None] * st["w_in"][1].double()      # (whole numbers first: a sum of 0 is 0)
    want = _silu(y[:, :inner]) * y[:, inner:]
    assert ((act.double() - want).abs() <= 1.01 * 2.0 ** -8 * want.abs() + 1e-5 * y[:, :inner].abs() * y[:, inner:].abs() + 1e-6 * want.abs()).all()
    q, s = _codes(act.double())
    assert torch.equal(qa, q)
    _same_scale(sa, s)
    want = (qa.double() @ st["w_down"][0].double().T) * sa.double()[:, None] * st["w_down"][1].double()
    assert ((out.double() - want).abs() <= 1.01 * 2.0 ** -8 * want.abs() + 4 * U * want.abs()).all()
    # two streams at the same time, each with operands of its own
    streams, runs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for stream in streams:
        with torch.cuda.stream(stream):
            mine = (x0.clone(), torch.empty_like(act), torch.empty_like(out))
            for _ in range(5):
                mine[0].copy_(x0)
                _feed_forward(st, mine[0], add, mine[2], mine[1], status)
            runs.append(mine)
    torch.cuda.synchronize()
    for mine in runs:
        assert torch.equal(mine[0], x) and torch.equal(mine[1], act) and torch.equal(mine[2], out)
    # captured twice, replayed with other inputs in between
    graphs, xs = [], []
    side = torch.cuda.Stream()
    for _ in range(2):
        gx, gact, gout = x0.clone(), torch.empty_like(act), torch.empty_like(out)
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=side):
                _feed_forward(st, gx, add, gout, gact, status)
        graphs.append(graph); xs.append((gx, gact, gout))
    for k in (0, 1, 0, 1):
        gx, gact, gout = xs[k]
        gx.normal_()
        graphs[k].replay()
        gx.copy_(x0)
        graphs[k].replay()
        torch.cuda.synchronize()
        assert torch.equal(gx, x) and torch.equal(gact, act) and torch.equal(gout, out)
    assert status.tolist() == [0, 0, 0, 0]


def test_offsets_beyond_32_bits():
    """Matrices of more than 2^31 entries: their last rows."""
    ops = _ops()
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    rows, width = 36000, 60000
    x = torch.zeros(rows, width, dtype=BF, device=DEV)
    x[-3:] = _x(3, width, BF)
    q, s = ops.q8_rows(rows, width, DEV), torch.empty(rows, device=DEV)
    ops.quantize_q8(q, s, x)
    want_q, want_s = _codes(x[-3:].double())
    assert torch.equal(q[-3:], want_q) and not q[:-3].any() and not s[:-3].any()
    _same_scale(s[-3:], want_s)
    ops.dequantize_q8(x, q, s)
    assert torch.equal(x[-3:], (q[-3:].float() * s[-3:, None]).bfloat16())
    gain = torch.ones(width, device=DEV)
    ops.rmsnorm_q8(q, s, x, gain, 1e-5, add=x, total=x)
    want_q = _codes((2 * (want_q.float() * want_s.float()[:, None]).bfloat16().double()))[0]
    assert torch.equal(q[-3:], want_q)
    del x, q
    T, N, K = 70000, 32768, 64
    a, sa, w, sw = _operands(T, N, K)
    for dtype, epilogue in ((BF, ops.EPILOGUE_STORE), (F32, ops.EPILOGUE_ACCUMULATE)):
        out = torch.zeros(T, N, dtype=dtype, device=DEV)
        ops.gemm_q8_tc(out, a, sa, w, sw, epilogue, status)
        want = (a[-40:].double() @ w.double().T) * sa[-40:].double()[:, None] * sw.double()
        assert ((out[-40:].double() - want).abs() <= (_half_step(dtype) * 1.01 + 4 * U) * want.abs()).all()
        del out
    assert status.tolist() == [0, 0, 0, 0]


def test_weights_made_by_the_kernel_in_front():
    """Rows that become integers just in front of the product that takes them as its weights, again and again over the same buffers: a product fetches its
    weights ahead of the kernel in front only where the caller says that they were there before."""
    ops = _ops()
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    for T, N, K in ((3, 2048, 4096), (600, 4096, 2048)):
        a, sa, _, _ = _operands(T, 1, K)
        w, sw = ops.q8_rows(N, K, DEV), torch.empty(N, device=DEV)
        xs = [torch.randn(N, K, device=DEV).bfloat16() for _ in range(4)]
        outs = [torch.empty(T, N, device=DEV) for _ in xs]
        for x, out in zip(xs, outs):
            ops.quantize_q8(w, sw, x)
            ops.gemm_q8_tc(out, a, sa, w, sw, ops.EPILOGUE_STORE, status)
        torch.cuda.synchronize()
        for x, out in zip(xs, outs):
            q, s = _codes(x.double())
            want = (a.double() @ q.double().T) * sa.double()[:, None] * s
            assert ((out.double() - want).abs() <= 6 * U * want.abs()).all()
    assert status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("tokens", [1, 61, 128, 700])
def test_products_of_both_kinds_follow_each_other(tokens):
    """bfloat16 and 8-bit products directly behind one another, eager and replayed: each has tensor memory of its own, and none waits for another's."""
    ops = _ops()
    K, N = 512, 1024
    status = ops.device_status(DEV)
    x, w = _x(tokens, K, BF, 3), (0.1 * torch.randn(N, K, device=DEV)).to(BF)
    (a, _), (b, _) = _fresh(tokens, K), _fresh(N, K)
    sa, sb = torch.empty(tokens, device=DEV), torch.empty(N, device=DEV)
    ops.quantize_q8(a, sa, x)
    ops.quantize_q8(b, sb, w)
    plain, short = torch.empty(tokens, N, dtype=BF, device=DEV), torch.empty(tokens, N, dtype=BF, device=DEV)

    def both():
        for _ in range(8):
            ops.gemm_tc(plain, x, w, ops.EPILOGUE_STORE, status)
            ops.gemm_q8_tc(short, a, sa, b, sb, ops.EPILOGUE_STORE, status, weights_settled=True)
    both()
    first = plain.clone(), short.clone()
    want = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    # two products with a scale, a conversion of a sum below 2^31: 4 half steps of float32, then one rounding to bfloat16
    assert ((first[1].double() - want).abs() <= (4 * U + _half_step(BF)) * 1.01 * want.abs()).all()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for _ in range(5):
        plain.zero_(), short.zero_()
        graph.replay()
        assert torch.equal(plain, first[0]) and torch.equal(short, first[1])
    assert int(status[0]) == 0
