"""The paged 8-bit key/value cache on the GPU: append bit for bit against exact arithmetic, the page operations against a
plain model, attention against 64 bits, and all of them together as a program uses them."""
import ctypes as C
import math

import numpy as np
import pytest

from tests import kv_model as M

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]


def say(text):
    print(text, flush=True)


def buf(a):
    from jxai_amd.moe import DeviceBuffer
    a = np.ascontiguousarray(a)
    return DeviceBuffer(a.nbytes).upload(a)


def code(name):
    from jxai_amd import formats as F
    return {"f32": F.F32, "f16": F.F16, "bf16": F.BF16}[name]


class Pair:
    """A cache on the GPU and its model on the host."""

    def __init__(self, layers=1, pages=16, P=64, H=2, D=64, seqs=4, most=8, seed=0):
        from jxai_amd import kv
        self.h = M.Cache(layers, pages, P, H, D, seqs, most)
        self.rng = np.random.default_rng(seed)
        # whatever was in the memory before
        self.h.codes[:] = self.rng.integers(-127, 128, self.h.codes.shape)
        self.h.scales[:] = self.rng.uniform(0.01, 0.03, self.h.scales.shape)
        self.h.table[:] = self.rng.integers(0, pages, self.h.table.shape)
        self.b = {n: buf(getattr(self.h, n)) for n in ("codes", "scales", "table", "len", "ref")}
        self.d = kv.KVCache(n_layers=layers, n_pages=pages, page_tokens=P, n_kv_heads=H, head_dim=D, max_seqs=seqs,
                            max_pages=most, buffers=self.b)

    def get(self, name):
        a = getattr(self.h, name)
        from jxai_amd._lib import lib
        assert lib().jx_device_synchronize() == 0
        return self.b[name].download(np.empty_like(a))

    def put(self, *names):
        for n in names:
            self.b[n].upload(getattr(self.h, n))

    def reserve(self, slots, n_new):
        s, n = buf(np.int32(slots)), buf(np.int32(n_new))
        self.d.reserve(s, n, len(slots))
        return self.h.reserve(slots, n_new)

    def check_books(self):
        assert self.d.status()[0] == 0
        assert np.array_equal(self.get("len"), self.h.len)
        assert np.array_equal(self.get("ref"), self.h.ref)
        assert np.array_equal(self.get("table"), self.h.table)

    def check_memory(self):
        assert np.array_equal(self.get("scales"), self.h.scales, equal_nan=True)
        assert np.array_equal(self.get("codes"), self.h.codes)

    def batch(self, slots, rows, max_len=0):
        from jxai_amd import kv
        start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.lists = (buf(np.int32(slots)), buf(start))
        return kv.KVBatch(n_seqs=len(slots), n_rows=int(start[-1]), max_rows=int(max(rows)), max_len=max_len, seqs=self.lists[0],
                          row_start=self.lists[1])

    def append(self, slots, rows, k, v, dtype, layer=0, strided=False):
        ka, kv_ = M.encode(k, dtype)
        va, vv = M.encode(v, dtype)
        H, D = self.h.H, self.h.D
        if strided:  # as two columns of one array, off 16-byte alignment
            wide = np.zeros((k.shape[0], 2 * H * D + 3), ka.dtype)
            wide[:, 1:1 + H * D] = ka.reshape(-1, H * D)
            wide[:, 2 + H * D:2 + 2 * H * D] = va.reshape(-1, H * D)
            b = buf(wide)
            at = b.ptr.value + ka.itemsize
            self.keep = b
            self.d.append(self.batch(slots, rows), at, at + (H * D + 1) * ka.itemsize, code(dtype), layer, wide.shape[1])
        else:
            self.keep = (buf(ka), buf(va))
            self.d.append(self.batch(slots, rows), *self.keep, code(dtype), layer)
        at = 0
        for s, n in zip(slots, rows):
            self.h.append(layer, s, kv_[at:at + n], vv[at:at + n])
            at += n

    def values(self, n, spread=1.0):
        H, D = self.h.H, self.h.D
        return (self.rng.standard_normal((2, n, H, D)) * spread).astype(np.float32)

    def attend(self, slots, rows, heads, dtype="f32", layer=0, max_len=0, sharp=1.0, scale=None, strided=False, ws=None, q=None,
               **how):
        from jxai_amd import kv
        from jxai_amd._lib import lib
        n, D = int(sum(rows)), self.h.D
        scale = scale or D ** -0.5
        if q is None:
            q = (self.rng.standard_normal((n, heads, D)) * sharp).astype(np.float32)
        qa, qv = M.encode(q, dtype)
        alibi = how.get("alibi")
        al = None if alibi is None else buf(np.float32(alibi))
        batch = self.batch(slots, rows, max_len)
        width = heads * D
        stride = width + 5 if strided else 0
        att = kv.Attention(n_heads=heads, dtype=code(dtype), scale=scale, softcap=how.get("softcap", 0.0),
                           window=how.get("window", 0), causal=how.get("causal", True), alibi=al, q_stride=stride,
                           out_stride=stride and width + 9)
        poison = np.full((n + 1, width + 9 if strided else width), {"f32": 7.0, "f16": 7.0, "bf16": 0x40E0}[dtype], qa.dtype)
        if strided:
            wide = np.zeros((n, stride), qa.dtype)
            wide[:, 1:1 + width] = qa.reshape(n, width)
            qb, ob = buf(wide), buf(poison)
            qp, op = qb.ptr.value + qa.itemsize, ob.ptr.value + 3 * qa.itemsize
        else:
            qb, ob = buf(qa), buf(poison)
            qp, op = qb, ob
        ws = self.d.workspace(batch, att) if ws is None else ws
        self.d.attend(batch, att, qp, op, ws, layer)
        assert lib().jx_device_synchronize() == 0
        got = ob.download(np.empty_like(poison))
        assert np.all(got[n] == poison[n])  # nothing behind the last row
        if strided:
            keep = np.ones(poison.shape, bool)
            keep[:n, 3:3 + width] = False
            assert np.all(got[keep] == poison[keep])
            got = got[:, 3:3 + width]
        out = M.decode(got[:n], dtype).reshape(n, heads, D)
        want, bound = M.attention(self.h, layer, slots, rows, qv, scale=scale, dtype=dtype,
                                  **{k: v for k, v in how.items() if k in ("softcap", "window", "causal", "alibi")})
        return out, want, bound


def near(out, want, bound):
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(out), nan)
    off, most = np.abs(out - want)[~nan], np.broadcast_to(bound, want.shape)[~nan]
    say(f"largest share of the bound: {(off / np.maximum(most, 1e-300)).max() if off.size else 0:.3f}")
    assert np.all(off <= most)  # where a row sees nothing, both are zero


def filled(D=64, H=2, P=64, lengths=(70, 1, 33), pages=64, dtype="f32", spread=1.0, seed=1, layers=1, most=None, rotate=True):
    """A cache whose slots hold tokens; its pages are out of order."""
    most = most or max(2, max(-(-n // P) for n in lengths) + 1)
    p = Pair(layers=layers, pages=pages, P=P, H=H, D=D, seqs=len(lengths) + 1, most=most, seed=seed)
    slots = [i for i, n in enumerate(lengths) if n]
    if rotate:  # holes: pages taken and given back
        p.h.ref[::3] = 1
        p.put("ref")
    assert p.reserve(slots, [lengths[i] for i in slots])
    if rotate:
        used = {int(x) for i in slots for x in p.h.table[i, :p.h.pages(lengths[i])]}
        p.h.ref[[x for x in range(0, pages, 3) if x not in used]] = 0
        p.put("ref")
    for layer in range(layers):
        k, v = p.values(sum(lengths), spread)
        p.append(slots, [lengths[i] for i in slots], k, v, dtype, layer)
    return p


# ------------------------------------------------------------------------------------------ append


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_append_pieces(D, dtype):
    """Pieces that begin and end inside a block, one token upwards, growing scales: bytes and scales as exact arithmetic."""
    p = Pair(P=64, H=3, D=D, seqs=3, pages=24, most=6, seed=D)
    for step, (slots, rows) in enumerate([([0, 2], [1, 40]), ([2, 0, 1], [1, 33, 64]), ([1, 0], [5, 1]), ([0, 1, 2], [30, 1, 95])]):
        say(f"append D={D} {dtype} step {step}")
        assert p.reserve(slots, rows)
        k, v = p.values(sum(rows), 1.0 + step)
        p.append(slots, rows, k, v, dtype, strided=step % 2 == 1)
    p.check_books()
    p.check_memory()


@pytest.mark.parametrize("P", [32, 128, 256])
def test_append_pages_and_layers(P):
    p = Pair(layers=3, P=P, H=1, D=64, seqs=2, pages=10, most=5, seed=P)
    for rows in ([P - 1, 2], [1, 1], [2, P]):
        assert p.reserve([1, 0], rows)
        for layer in (2, 0):
            k, v = p.values(sum(rows))
            p.append([1, 0], rows, k, v, "f32", layer)
    p.check_books()
    p.check_memory()


def test_append_special_values():
    """Zeros, the middle of two codes, the smallest and largest values, values that are not finite."""
    p = Pair(P=32, H=1, D=32, seqs=8, pages=16, most=2, seed=3)
    k, v = p.values(32)
    v[:] = 0  # block of zeros
    # exact middles: scale 2^-7 * 127 / 127
    k[:, 0] = (p.rng.integers(-254, 255, (32, 32)) / 2).astype(np.float32)
    k[0, 0, 0] = 127.0
    assert p.reserve([0], [32])
    p.append([0], [32], k, v, "f32")
    cases = [1e-45, 2.0 ** -126, 2.0 ** -119, 3.0e38, np.inf, np.nan]
    for slot, x in enumerate(cases, 1):
        assert p.reserve([slot], [3])
        k, v = p.values(3)
        k *= np.float32(min(abs(x), 1.0) if np.isfinite(x) else 1.0)
        k[1, 0, 5] = x
        v[2, 0, 31] = -x
        p.append([slot], [3], k, v, "f32")
    for slot, x in enumerate(cases, 1):  # behind them
        assert p.reserve([slot], [2])
        k, v = p.values(2)
        p.append([slot], [2], k, v, "f32")
    p.check_books()
    assert np.array_equal(p.get("scales"), p.h.scales, equal_nan=True)
    fine = ~np.isnan(p.h.scales)
    assert np.array_equal(p.get("codes")[fine], p.h.codes[fine])


def test_append_middles():
    """Quotients next to the middle of two codes, where a product with the reciprocal rounds to the wrong side."""
    p = Pair(P=256, H=1, D=256, seqs=1, pages=2, most=2, seed=4)
    k, v = p.values(256)
    for x in (k, v):
        for b in range(0, 256, 32):
            top = np.float32(p.rng.uniform(1, 2))
            s = np.float32(top / np.float32(127))
            mid = (p.rng.integers(-127, 127, (32, 256)) + 0.5) * np.float64(s)
            m = mid.astype(np.float32)
            x[b:b + 32, 0] = np.nextafter(m, np.where(p.rng.integers(0, 2, m.shape), np.float32(np.inf), np.float32(-np.inf)).astype(np.float32))
            x[b:b + 32, 0, ::3] = m[:, ::3]
            np.clip(x[b:b + 32, 0], -top, top, out=x[b:b + 32, 0])
            x[b, 0, 0] = top
    assert p.reserve([0], [256])
    p.append([0], [256], k, v, "f32")
    p.check_memory()


# ------------------------------------------------------------------------------------------ pages


def test_pages_random_program():
    """A few hundred page operations in random order, three layers."""
    p = Pair(layers=3, pages=40, P=32, H=1, D=32, seqs=9, most=7, seed=11)
    r = p.rng
    for step in range(300):
        op = r.choice(["reserve", "reserve", "trim", "fork", "fork", "compact", "append"])
        n = int(r.integers(1, 6))
        slots = [int(x) for x in r.permutation(9)[:n]]
        if op == "reserve":
            new = [int(r.integers(0, 1 + min(70, 7 * 32 - p.h.len[s]))) for s in slots]
            if not p.reserve(slots, new):
                assert p.d.status()[0] == 4
                with pytest.raises(Exception, match="free pages"):
                    p.d.check_status()
        elif op == "trim":
            to = [int(r.integers(-1, 1 + p.h.len[s])) if r.random() < 0.6 else 0 for s in slots]
            need = sum(1 for t in to if t > 0)
            if len(p.h.free()) < need:
                continue
            p.d.trim(buf(np.int32(slots)), buf(np.int32(to)), n)
            p.h.trim(slots, to)
        elif op == "fork":
            src = [int(x) for x in r.integers(0, 9, n)]
            if len(p.h.free()) < n:
                continue
            p.d.fork(buf(np.int32(src)), buf(np.int32(slots)), n)
            p.h.fork(src, slots)
        elif op == "compact":
            p.d.compact()
            assert p.h.compact() == p.d.status()[1]
        else:
            # a full last page may be shared: then the append is refused (test_append_into_a_shared_page)
            slots = [s for s in slots if p.h.len[s] > 0 and p.h.ref[p.h.table[s, (p.h.len[s] - 1) // 32]] == 1]
            own = [min(3, int(p.h.len[s] - 1) % 32 + 1) for s in slots]  # within the last page, which is the slot's own
            if slots:
                k, v = p.values(sum(own))
                p.append(slots, own, k, v, "f32", int(r.integers(0, 3)))
        if step % 10 == 9:
            say(f"pages: step {step} {op}, {int((p.h.ref > 0).sum())} pages in use")
            p.check_books()
            p.check_memory()


def test_append_into_a_shared_page():
    """After a fork at a page's end both slots hold the last page: writing its tokens again is refused, and so for earlier ones."""
    p = filled(D=64, H=1, P=32, lengths=(64, 0, 0), pages=12, most=4, rotate=False)
    p.d.fork(buf(np.int32([0])), buf(np.int32([1])), 1)
    p.h.fork([0], [1])
    for slot in (0, 1):
        k, v = p.values(3)
        kb = (buf(k), buf(v))
        p.d.append(p.batch([slot], [3]), *kb)
        assert p.d.status()[0] == 8
        with pytest.raises(Exception, match="another slot"):
            p.d.check_status()
        p.check_books()
        p.check_memory()
    assert p.reserve([1], [2])  # a page of its own behind them
    k, v = p.values(2)
    p.append([1], [2], k, v, "f32")
    p.check_books()
    p.check_memory()


def test_pages_many():
    """More slots, list entries and pages than the bookkeeping's workgroup has threads."""
    p = Pair(pages=9000, P=32, H=1, D=32, seqs=1500, most=5, seed=12)
    every = [int(x) for x in p.rng.permutation(1500)[:1400]]
    assert p.reserve(every, [int(x) for x in p.rng.integers(1, 140, 1400)])
    p.check_books()
    gone = every[::2]
    p.d.trim(buf(np.int32(gone)), None, len(gone))
    p.h.trim(gone, [0] * len(gone))
    src = [int(x) for x in p.rng.choice(every[1::2], 600)]
    dst = gone[:600]
    p.d.fork(buf(np.int32(src)), buf(np.int32(dst)), 600)
    p.h.fork(src, dst)
    p.check_books()
    p.d.compact()
    p.h.compact()
    p.check_books()
    p.check_memory()


def test_pages_refuse_on_the_device():
    """What only the device can see: reported, and nothing changed."""
    p = filled(D=32, H=1, P=32, lengths=(40, 70, 1), pages=9, most=4, rotate=False)
    i32 = lambda *v: buf(np.int32(v))  # noqa: E731
    calls = {
        "twice": lambda: p.d.trim(i32(1, 0, 1), None, 3),
        "slot": lambda: p.d.trim(i32(4), None, 1),
        "negative slot": lambda: p.d.fork(i32(0), i32(-1), 1),
        "source": lambda: p.d.fork(i32(9), i32(3), 1),
        "too long": lambda: p.d.reserve(i32(0), i32(4 * 32 - 39), 1),
        "negative": lambda: p.d.reserve(i32(0), i32(-1), 1),
        "pages": lambda: p.d.reserve(i32(0, 2, 3), i32(60, 60, 60), 3),
        "pages of a fork": lambda: (p.d.reserve(i32(3), i32(96), 1), p.h.reserve([3], [96]),
                                    p.d.fork(i32(0, 1), i32(3, 2), 2)),
    }
    for name, call in calls.items():
        say(f"refusal: {name}")
        call()
        bits = p.d.status()[0]
        assert bits == (4 if name.startswith("pages") else 2), name
        # nothing runs until the program has looked
        p.d.trim(i32(0), None, 1)
        p.d.compact()
        k, v = p.values(1)
        kb = (buf(k), buf(v))
        p.d.append(p.batch([0], [1]), *kb)
        assert np.isnan(p.attend([0], [1], 2)[0]).all()
        with pytest.raises(Exception, match="KVCache"):
            p.d.check_status()
        p.check_books()
        p.check_memory()


def test_bad_pages_and_rows():
    """Table entries outside the cache and rows outside their limits: NaN or untouched rows, a bit, no access outside."""
    p = filled(D=64, H=2, P=32, lengths=(70, 40, 33), pages=12, most=4, rotate=False)
    good = p.h.table.copy()
    for bad in (-1, 12, 2 ** 31 - 1, -2 ** 31):
        p.h.table[:] = good
        p.h.table[0, 1] = bad
        p.put("table")
        p.h.table[0, 1] = 0
        out, want, bound = p.attend([0, 1], [1, 1], 2)
        assert np.isnan(out[0]).all()
        assert p.d.status()[0] == 1
        with pytest.raises(Exception, match="no page"):
            p.d.check_status()
        p.h.table[:] = good
        p.h.table[2, 1] = bad
        p.put("table")
        k, v = p.values(2)
        kb = (buf(k), buf(v))
        p.d.append(p.batch([2], [2]), *kb)  # one row into the good page 0, one into the bad one
        assert p.d.status()[0] == 1
        p.d.trim(buf(np.int32([2])), buf(np.int32([1])), 1)
        with pytest.raises(Exception, match="no page"):
            p.d.check_status()
        p.d.trim(buf(np.int32([2])), buf(np.int32([1])), 1)
        assert p.d.status()[0] == 1
        with pytest.raises(Exception, match="no page"):
            p.d.check_status()
    p.h.table[:] = good
    p.put("table")
    from jxai_amd import kv
    q, o = buf(np.ones((8, 2, 64), np.float32)), buf(np.full((8, 2, 64), 7, np.float32))
    att = kv.Attention(n_heads=2, scale=0.1)
    for name, seqs, start, most in (("slot", [9], [0, 1], 1), ("order", [0], [2, 1], 1), ("behind", [0], [0, 9], 8),
                                    ("many", [0], [0, 3], 2), ("negative", [0], [-1, 0], 1)):
        say(f"rows: {name}")
        lists = buf(np.int32(seqs)), buf(np.int32(start))
        b = kv.KVBatch(n_seqs=1, n_rows=8, max_rows=most, seqs=lists[0], row_start=lists[1])
        p.d.attend(b, att, q, o, p.d.workspace(b, att))
        assert p.d.status()[0] == 2
        assert np.all(o.download(np.empty((8, 2, 64), np.float32)) == 7)
        with pytest.raises(Exception, match="limits"):
            p.d.check_status()
        p.d.append(b, q, q)
        assert p.d.status()[0] == 2
        with pytest.raises(Exception, match="limits"):
            p.d.check_status()
    p.d.append(p.batch([1], [41]), buf(np.zeros((41, 2, 64), np.float32)), buf(np.zeros((41, 2, 64), np.float32)))  # more rows than tokens
    assert p.d.status()[0] == 2
    with pytest.raises(Exception, match="limits"):
        p.d.check_status()


# ------------------------------------------------------------------------------------------ attention


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_single_rows(D, dtype):
    """One row per sequence, from one token to a few pages; groups of heads of every size up to more than a tile's rows."""
    for seed, (H, G, P) in enumerate([(2, 1, 64), (1, 4, 32), (3, 7, 128), (1, 40, 64)]):
        lengths = (1, 31, 32, 33, 0, 64, 65, 200, 500)
        p = filled(D=D, H=H, P=P, lengths=lengths, pages=90, seed=seed + D)
        say(f"attend D={D} {dtype} H={H} G={G} P={P}")
        slots = [8, 0, 1, 2, 4, 3, 5, 6, 7]  # slot 4 is empty
        near(*p.attend(slots, [1 if p.h.len[s] else 0 for s in slots], H * G, dtype, sharp=2.0, strided=seed % 2 == 1))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [(2, 5, 1), (33, 64, 17), (100, 0, 257), (300, 1, 31)])
def test_attend_many_rows(D, dtype, rows):
    lengths = tuple(n + e for n, e in zip(rows, (0, 70, 129)))
    p = filled(D=D, H=2, P=64, lengths=lengths, pages=40, seed=sum(rows))
    say(f"attend rows={rows} D={D} {dtype}")
    near(*p.attend([0, 1, 2], list(rows), 6, dtype, max_len=max(lengths)))


@pytest.mark.parametrize("how", [dict(window=1), dict(window=40), dict(window=1000), dict(softcap=5.0), dict(softcap=30.0, window=33),
                                 dict(causal=False), dict(causal=False, window=64), dict(alibi=True),
                                 dict(alibi=True, softcap=20.0, causal=False), dict(alibi=True, window=50)],
                         ids=lambda h: "-".join(f"{k}{v}" for k, v in h.items()))
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_masks(how, dtype):
    how = dict(how)
    if how.get("alibi"):
        how["alibi"] = [0.5, 0.25, 0.0, -0.01]
    for D, rows in ((64, (1, 1, 1)), (128, (5, 1, 40)), (96, (150, 70, 33))):
        p = filled(D=D, H=2, P=32, lengths=(151, 130, 33), pages=60, seed=D)
        say(f"masks {how} {dtype} D={D} rows={rows}")
        near(*p.attend([0, 1, 2], list(rows), 4, dtype, sharp=3.0, **how))


def test_attend_more_rows_than_tokens():
    """Rows before the first token see nothing: zeros."""
    p = filled(D=64, H=1, P=32, lengths=(3, 40), pages=8)
    out, want, bound = p.attend([0, 1], [9, 2], 2)
    assert np.all(out[:6] == 0) and np.all(want[:6] == 0)
    near(out, want, bound)
    p.h.len[0] = 0
    p.put("len")
    for causal in (True, False):
        out, want, bound = p.attend([0, 1], [2, 1], 2, causal=causal)
        assert np.all(out[:2] == 0)
        near(out, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,H,G", [(128, 1, 1), (64, 2, 4), (256, 1, 2)])
def test_attend_long(D, H, G, dtype):
    """A long axis for few rows: divided and joined; the hint about the longest sequence too small, exact, unknown."""
    n = 9000
    p = filled(D=D, H=H, P=128, lengths=(n, 77), pages=90, seed=5, rotate=False)
    for max_len in (n, 0, 300):
        for rows in ([1, 1], [3, 2]):
            say(f"long D={D} H={H} G={G} {dtype} max_len={max_len} rows={rows}")
            near(*p.attend([0, 1], rows, H * G, dtype, max_len=max_len, sharp=3.0))
    near(*p.attend([0, 1], [1, 1], H * G, dtype, window=5000))


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attend_uneven_batches(D, dtype):
    """Few rows over sequences of very different lengths, 1 to 32 rows times heads, more sequences than a wave has lanes."""
    for G, rows, lengths in ((1, 1, (1, 1500, 0, 37, 2300, 64)), (5, 3, (40, 1100, 2000, 7)), (16, 1, (1700, 3)), (17, 1, (1300, 90)),
                             (4, 8, (8, 1200, 600)), (2, 1, tuple(int(x) for x in np.random.default_rng(D).integers(0, 300, 70)) + (1200,))):
        p = filled(D=D, H=2, P=64, lengths=lengths, pages=260, seed=D + G, rotate=False)
        say(f"uneven D={D} {dtype} G={G} rows={rows} sequences={len(lengths)}")
        slots = list(range(len(lengths)))[::-1]
        near(*p.attend(slots, [min(rows, lengths[s]) for s in slots], 2 * G, dtype, sharp=2.0, strided=G == 5))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_scales_apart(dtype):
    """Blocks whose scales lie far apart, zero blocks among them, in every order: weights stay in range."""
    for order in (1, -1, 7):
        p = Pair(P=32, H=2, D=64, seqs=1, pages=20, most=20, seed=order + 9)
        sizes = [1e-30, 1e-6, 1.0, 0.0, 1e4, 1e20][::order] if abs(order) == 1 else [1.0, 1e-10, 1e10, 0.0, 1e-3, 1e-3]
        for s in sizes:
            assert p.reserve([0], [32])
            k, v = p.values(32)
            p.append([0], [32], k, v * np.float32(s), "f32")
        say(f"scales {sizes} {dtype}")
        near(*p.attend([0], [3], 4, dtype))


def test_attend_large_scores():
    """Scores far apart, and rows of very small and large q."""
    p = filled(D=64, H=1, P=32, lengths=(300,), pages=20, seed=8)
    for sharp in (1e-20, 1e-3, 300.0, 1e5):
        say(f"scores {sharp}")
        near(*p.attend([0], [4], 2, "f32", sharp=sharp))


def test_attend_not_finite():
    """A row of q that is not finite gives NaN, other rows nothing of it; a block that reads as NaN reaches the rows that see it."""
    p = filled(D=64, H=1, P=32, lengths=(100,), pages=20, seed=8)
    for bad in (np.nan, np.inf, -np.inf):
        q = p.rng.standard_normal((40, 2, 64)).astype(np.float32)
        q[3, 1, 7] = bad
        for rows, dtype in (([40], "f32"), ([40], "bf16")):
            out, want, bound = p.attend([0], rows, 2, dtype, q=q)
            assert np.isnan(out[3, 1]).all()
            fine = np.ones((40, 2), bool)
            fine[3, 1] = False
            near(out[fine], want[fine], np.broadcast_to(bound, want.shape)[fine])
    assert p.reserve([0], [1])
    k, v = p.values(1)
    v[0, 0, 3] = np.nan
    p.append([0], [1], k, v, "f32")
    for dtype in ("f32", "f16"):
        out, want, bound = p.attend([0], [20], 2, dtype)  # tokens 81 .. 100: the block 96 .. 127 is NaN
        assert np.isnan(out[15:]).all()
        assert np.isfinite(out[:15]).all()
        near(out[:15], want[:15], bound[:15])


def test_attend_in_place_and_repeatable():
    """out over q; the same bits on every call."""
    from jxai_amd import kv
    from jxai_amd._lib import lib
    p = filled(D=128, H=2, P=64, lengths=(700, 3000), pages=70, seed=21, rotate=False)
    q = p.rng.standard_normal((2, 8, 128)).astype(np.float32)
    att, batch = kv.Attention(n_heads=8, scale=0.1), p.batch([0, 1], [1, 1], 3000)
    ws = p.d.workspace(batch, att)
    first = None
    for i in range(20):
        b = buf(q)
        p.d.attend(batch, att, b, b, ws)
        assert lib().jx_device_synchronize() == 0
        got = b.download(np.empty_like(q))
        first = got if first is None else first
        assert np.array_equal(first, got)
    want, bound = M.attention(p.h, 0, [0, 1], [1, 1], q, scale=0.1)
    near(first.astype(np.float64), want, bound)


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB: the last page and layer."""
    p_tokens, H, D = 256, 8, 128
    page = 2 * H * p_tokens * D
    pages = (5 << 30) // page
    from jxai_amd import kv
    from jxai_amd._lib import lib
    d = kv.KVCache(n_layers=1, n_pages=pages, page_tokens=p_tokens, n_kv_heads=H, head_dim=D, max_seqs=1, max_pages=4)
    table = np.int32([[pages - 1, 0, pages - 2, 5]])
    d.buffers["table"].upload(table)
    d.buffers["len"].upload(np.int32([600]))
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((2, 600, H, D)).astype(np.float32)
    h = M.Cache(1, 4, p_tokens, H, D, 1, 4)
    h.table[:] = [[0, 1, 2, 3]]
    h.len[:] = 600
    h.append(0, 0, k, v)
    start = buf(np.int32([0, 600]))
    kb, vb = buf(k), buf(v)
    d.append(kv.KVBatch(n_seqs=1, n_rows=600, max_rows=600, row_start=start), kb, vb)
    q = rng.standard_normal((1, 16, D)).astype(np.float32)
    qb, ob = buf(q), buf(np.zeros_like(q))
    batch, att = kv.KVBatch(n_seqs=1), kv.Attention(n_heads=16, scale=D ** -0.5)
    d.attend(batch, att, qb, ob, d.workspace(batch, att))
    assert d.status()[0] == 0
    want, bound = M.attention(h, 0, [0], [1], q, scale=D ** -0.5)
    near(ob.download(np.empty_like(q)).astype(np.float64), want, bound)
    assert lib().jx_device_synchronize() == 0


# ------------------------------------------------------------------------------------------ together


def test_graph_of_a_step():
    """A decode step (reserve, append, attend) captured once and replayed, with the program's own work between the replays."""
    from jxai_amd import kv
    from jxai_amd._lib import lib
    hip = C.CDLL("libamdhip64.so")
    p = filled(D=64, H=2, P=32, lengths=(30, 61, 5), pages=40, most=8, seed=31, layers=2)
    slots, n = [2, 0, 1], 3
    s = buf(np.int32(slots))
    batch = kv.KVBatch(n_seqs=n, max_len=200, seqs=s)
    att = kv.Attention(n_heads=8, scale=0.125)
    ws = p.d.workspace(batch, att)
    kb, vb, qb = (buf(np.zeros((n, w, 64), np.float32)) for w in (2, 2, 8))
    ob = [buf(np.zeros((n, 8, 64), np.float32)) for _ in range(2)]
    st = C.c_void_p()
    assert hip.hipStreamCreate(C.byref(st)) == 0
    assert hip.hipStreamBeginCapture(st, 1) == 0
    p.d.reserve(s, None, n, st.value)
    for layer in range(2):
        p.d.append(batch, kb, vb, layer=layer, stream=st.value)
        p.d.attend(batch, att, qb, ob[layer], ws, layer, st.value)
    g, ex = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamEndCapture(st, C.byref(g)) == 0
    assert hip.hipGraphInstantiate(C.byref(ex), g, None, None, 0) == 0
    for i in range(12):
        say(f"graph: replay {i}")
        k, v = p.values(n, 1 + i % 3)
        q = p.rng.standard_normal((n, 8, 64)).astype(np.float32)
        kb.upload(k), vb.upload(v), qb.upload(q)
        assert hip.hipGraphLaunch(ex, st) == 0
        assert hip.hipStreamSynchronize(st) == 0
        p.h.reserve(slots, [1] * n)
        for layer in range(2):
            for j, slot in enumerate(slots):
                p.h.append(layer, slot, k[j:j + 1], v[j:j + 1])
            want, bound = M.attention(p.h, layer, slots, [1] * n, q, scale=0.125)
            near(ob[layer].download(np.empty_like(q)).astype(np.float64), want, bound)
        if i % 4 == 3:  # the program's own work between
            p.d.compact()
            p.h.compact()
        p.check_books()
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(g)
    hip.hipStreamDestroy(st)
    p.check_memory()
    assert lib().jx_device_synchronize() == 0


def test_two_streams_read_at_once():
    """Two attentions of one cache on two streams, each with a workspace of its own."""
    from jxai_amd import kv
    hip = C.CDLL("libamdhip64.so")
    p = filled(D=128, H=2, P=64, lengths=(5000, 4000), pages=160, seed=41, rotate=False)
    calls = []
    for slot in (0, 1):
        st = C.c_void_p()
        assert hip.hipStreamCreate(C.byref(st)) == 0
        q = p.rng.standard_normal((1, 8, 128)).astype(np.float32)
        s = buf(np.int32([slot]))
        batch, att = kv.KVBatch(n_seqs=1, max_len=5000, seqs=s), kv.Attention(n_heads=8, scale=0.1)
        calls.append((st, q, s, batch, att, buf(q), buf(np.zeros_like(q)), p.d.workspace(batch, att), slot))
    for _ in range(10):
        for st, q, s, batch, att, qb, ob, ws, slot in calls:
            p.d.attend(batch, att, qb, ob, ws, stream=st.value)
    for st, q, s, batch, att, qb, ob, ws, slot in calls:
        assert hip.hipStreamSynchronize(st) == 0
        want, bound = M.attention(p.h, 0, [slot], [1], q, scale=0.1)
        near(ob.download(np.empty_like(q)).astype(np.float64), want, bound)
        hip.hipStreamDestroy(st)


def test_generation_with_a_layer():
    """The set as a program uses it: a prompt through the q/k/v projection's products into the cache, answers forked from
    it, steps of projection, append and attention, the MoE layer behind; a sequence that generates alone agrees with the same
    tokens in one piece."""
    from jxai_amd import formats as F
    from jxai_amd import kv, moe, synth
    from jxai_amd._lib import check, lib
    moe.init(0)
    cfg = synth.CONFIGS["toy"]
    d, H, G, D = cfg.d_model, 2, 4, 64
    rng = np.random.default_rng(3)

    def matrix(rows):
        blk, size = F.BLOCK[F.Q8_0]
        raw = np.zeros((rows * d // blk, size), np.uint8)
        raw[:, :2] = (0.002 + 0.004 * rng.random(len(raw))).astype(np.float16).view(np.uint8).reshape(-1, 2)
        raw[:, 2:] = rng.integers(-127, 128, (len(raw), 32)).astype(np.int8).view(np.uint8)
        return moe.QMatrix(F.Q8_0, raw.reshape(-1), rows, d)

    wq, wk, wv, wo = matrix(H * G * D), matrix(H * D), matrix(H * D), matrix(d) if H * G * D == d else None
    layer = moe.MoELayer.from_weights(synth.make_layer(cfg))
    p = Pair(P=32, H=H, D=D, seqs=4, pages=30, most=6, seed=5)
    x = rng.standard_normal((50, d)).astype(np.float32)
    xb, qb = buf(x), buf(np.zeros((50, H * G * D), np.float32))
    kb, vb = buf(np.zeros((50, H * D), np.float32)), buf(np.zeros((50, H * D), np.float32))

    def project(n):
        for i in range(n):
            at = [C.c_void_p(b.ptr.value + 4 * i * w) for b, w in ((xb, d), (qb, H * G * D), (kb, H * D), (vb, H * D))]
            check(lib().jx_matmul_qkv_quant_f32_dev(wq.handle, wk.handle, wv.handle, *at, None), "qkv")

    att = kv.Attention(n_heads=H * G, scale=D ** -0.5)
    ob, mb = buf(np.zeros((50, H * G * D), np.float32)), buf(np.zeros((50, d), np.float32))

    def pull(b, n, w):
        check(lib().jx_device_synchronize(), "sync")
        return b.download(np.empty((50, w), np.float32))[:n]

    def step(slots, rows):
        n = sum(rows)
        project(n)
        assert p.reserve(slots, rows)
        batch = p.batch(slots, rows)
        p.d.append(batch, kb, vb)
        k, v = pull(kb, n, H * D).reshape(n, H, D), pull(vb, n, H * D).reshape(n, H, D)
        at = 0
        for s, m in zip(slots, rows):
            p.h.append(0, s, k[at:at + m], v[at:at + m])
            at += m
        p.d.attend(batch, att, qb, ob, p.d.workspace(batch, att))
        q = pull(qb, n, H * G * D).reshape(n, H * G, D)
        want, bound = M.attention(p.h, 0, slots, rows, q, scale=D ** -0.5)
        near(pull(ob, n, H * G * D).reshape(n, H * G, D).astype(np.float64), want, bound)
        if H * G * D == d:  # the layer behind takes the attention's rows where they lie
            layer.forward_device(ob, n, mb)
            out, _, _, _ = layer.forward(pull(ob, n, d))
            assert np.array_equal(out, pull(mb, n, d))

    step([0], [45])
    p.d.fork(buf(np.int32([0, 0])), buf(np.int32([1, 3])), 2)
    p.h.fork([0, 0], [1, 3])
    p.check_books()
    for i in range(4):
        xb.upload(np.concatenate([rng.standard_normal((3, d)).astype(np.float32), x[3:]]))
        step([1, 0, 3], [1, 1, 1])
    p.d.trim(buf(np.int32([3])), buf(np.int32([40])), 1)  # back into what is shared
    p.h.trim([3], [40])
    step([3, 1], [7, 2])
    p.d.trim(buf(np.int32([0])), None, 1)
    p.h.trim([0], [0])
    p.d.compact()
    p.h.compact()
    step([1, 3], [1, 4])
    p.check_books()
    p.check_memory()
    layer.close()
