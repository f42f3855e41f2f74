"""laya_op_attend and laya_op_document_bounds on the GPU against 64 bits (bounds: attend_reference.py)."""
import ctypes as ct

import numpy as np
import pytest

import attend_reference as A
from laya_cuda import _lib

pytestmark = pytest.mark.gpu

CODE = {"f16": _lib.F16, "bf16": _lib.BF16}


def torch():
    import torch as t
    return t


def at(x):
    return None if x is None else x.data_ptr()


class Call:
    """Packed sequences with gaps between them, their inputs on the device, the call, and the same in 64 bits."""

    def __init__(self, gpu, kind, lengths, heads, kv_heads, dim, *, key_lengths=None, cap=0.0, bias=None, span=0, before=-1, after=-1,
                 prefix=False, documents=False, scale=None, seed=0, size=1.5, gap=3, extra=8):
        t = torch()
        rng = np.random.default_rng(seed)
        self.kind, self.heads, self.kv_heads, self.dim, self.gpu = kind, heads, kv_heads, dim, gpu
        self.nq = np.array(lengths, np.int32)
        self.nk = np.array(lengths if key_lengths is None else key_lengths, np.int32)
        self.q0 = (np.cumsum(self.nq + gap) - self.nq).astype(np.int32)
        self.k0 = (np.cumsum(self.nk + gap) - self.nk).astype(np.int32)
        q_rows, k_rows = int(self.nq.sum() + gap * len(self.nq) + gap), int(self.nk.sum() + gap * len(self.nk) + gap)
        dtype = {"f16": t.float16, "bf16": t.bfloat16}[kind]
        # Heads lie `extra` values further apart than they are wide; what is between them and in rows of no sequence is NaN.
        self.q = t.full((q_rows, heads, dim + extra), float("nan"), dtype=dtype, device=gpu)
        self.kv = t.full((k_rows, 2 * kv_heads, dim + extra), float("nan"), dtype=dtype, device=gpu)
        for s in range(len(self.nq)):
            self.q[self.q0[s]:self.q0[s] + self.nq[s], :, :dim] = t.from_numpy(rng.normal(0, size, (self.nq[s], heads, dim))).to(gpu).to(dtype)
            self.kv[self.k0[s]:self.k0[s] + self.nk[s], :, :dim] = t.from_numpy(rng.normal(0, 1, (self.nk[s], 2 * kv_heads, dim))).to(gpu).to(dtype)
        self.out = t.full((q_rows, heads, dim + extra), 9.0, dtype=dtype, device=gpu)
        self.scale = float(np.float32(dim ** -0.5 if scale is None else scale))
        self.cap, self.before, self.after = float(np.float32(cap)), before, after
        self.slopes = (np.exp2(-8.0 * np.arange(1, heads + 1) / heads) * rng.uniform(.5, 1.5, heads)).astype(np.float32) if bias == "slopes" else None
        self.table = rng.normal(0, 1.5, (heads, 2 * span + 1)).astype(np.float32) if bias == "table" else None
        self.span = span
        self.prefix = np.array([rng.integers(0, n + 1) // 3 for n in self.nk], np.int32) if prefix else None
        self.bounds = None
        if documents:
            self.bounds = np.full((q_rows, 2), -7, np.int32)
            for s, n in enumerate(self.nq):
                ids = np.cumsum(rng.random(self.nk[s]) < .03)
                self.bounds[self.q0[s]:self.q0[s] + n] = A.document_bounds(ids)[self.nk[s] - n:]
        self.workspace = None

    def up(self, x):
        return None if x is None else torch().from_numpy(x).to(self.gpu)

    def describe(self, **change):
        self.kept = {name: self.up(getattr(self, name)) for name in ("q0", "nq", "k0", "nk", "prefix", "bounds", "slopes", "table")}
        d = self.kept
        values = dict(struct_bytes=ct.sizeof(_lib.LayaAttend), dtype=CODE[self.kind], q=at(self.q), k=at(self.kv),
                      v=self.kv.data_ptr() + 2 * self.kv_heads * self.kv.stride(1), out=at(self.out), q_row=self.q.stride(0),
                      q_head=self.q.stride(1), k_row=self.kv.stride(0), k_head=self.kv.stride(1), v_row=self.kv.stride(0),
                      v_head=self.kv.stride(1), out_row=self.out.stride(0), out_head=self.out.stride(1), heads=self.heads,
                      kv_heads=self.kv_heads, dim=self.dim, q_rows=self.q.shape[0], k_rows=self.kv.shape[0], n_seq=len(self.nq),
                      max_q=int(self.nq.max(initial=0)), max_k=int(self.nk.max(initial=0)), q_starts=at(d["q0"]), q_lengths=at(d["nq"]),
                      k_starts=at(d["k0"]), k_lengths=at(d["nk"]), scale=self.scale, cap=self.cap, slopes=at(d["slopes"]),
                      table=at(d["table"]), span=self.span, before=self.before, after=self.after, prefix=at(d["prefix"]),
                      bounds=at(d["bounds"]))
        self.call = _lib.LayaAttend(**{**values, **change})
        need = _lib.load().laya_attend_workspace(ct.byref(self.call))
        assert need >= 0
        self.workspace = torch().full((max(need, 16),), 0xff, dtype=torch().uint8, device=self.gpu) if need else None  # NaNs
        return self

    def run(self, stream=None):
        stream = stream or torch().cuda.current_stream()
        size = 0 if self.workspace is None else self.workspace.numel()
        _lib.check(_lib.load().laya_op_attend(ct.byref(self.call), at(self.workspace), size, ct.c_void_p(stream.cuda_stream)))
        return self

    def expected(self):
        q, kv = self.q.double().cpu().numpy(), self.kv.double().cpu().numpy()
        out = np.full(self.out.shape, 9.0)
        bound = np.zeros(self.out.shape)
        for s in range(len(self.nq)):
            rows = slice(self.q0[s], self.q0[s] + self.nq[s])
            keys = slice(self.k0[s], self.k0[s] + self.nk[s])
            out[rows, :, :self.dim], bound[rows, :, :self.dim] = A.attend(
                q[rows, :, :self.dim], kv[keys, :self.kv_heads, :self.dim], kv[keys, self.kv_heads:, :self.dim], self.scale, self.cap,
                self.slopes, self.table, self.before, self.after, 0 if self.prefix is None else self.prefix[s],
                None if self.bounds is None else self.bounds[rows], self.kind)
        return out, bound

    def check(self):
        torch().cuda.synchronize()
        got = self.out.double().cpu().numpy()
        want, bound = self.expected()
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        off = np.abs(got - want)[~np.isnan(want)] - bound[~np.isnan(want)]
        assert not np.isnan(off).any() and off.max(initial=0) <= 0, (off.max(), np.abs(got - want)[~np.isnan(want)].max())
        return self


ODD = [1, 0, 63, 64, 65, 127, 128, 129, 31, 200, 33]
KERNELS = pytest.mark.parametrize("kernel", [_lib.ATTEND_MANY, _lib.ATTEND_FEW], ids=["many", "few"])
BIASES = [("none", None, 0), ("slopes", "slopes", 0), ("table", "table", 20)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 96, 104, 128, 136, 160, 168, 192, 200, 256])
@KERNELS
def test_widths(gpu, kind, dim, kernel):
    Call(gpu, kind, ODD, 4, 2, dim).describe(kernel=kernel).run().check()


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("n", [1, 60, 300])
def test_planned(gpu, dim, n):
    """The planner's choice, from few rows to more sequences than lanes and than one round of workgroups."""
    Call(gpu, "bf16", ODD[:6] + [17] * n, 4, 4, dim, after=0).describe().run().check()


@pytest.mark.parametrize("kind,dim", [("f16", 64), ("bf16", 128), ("f16", 96), ("bf16", 256), ("f16", 192)])
@pytest.mark.parametrize("cap", [0.0, 7.0])
@pytest.mark.parametrize("bias,span", [b[1:] for b in BIASES], ids=[b[0] for b in BIASES])
@pytest.mark.parametrize("masks", [dict(), dict(after=0), dict(before=37, after=5), dict(after=0, prefix=True),
                                   dict(prefix=True, documents=True), dict(documents=True, before=20)],
                         ids=["all", "causal", "window", "prefix", "documents", "near"])
@KERNELS
def test_masks_caps_and_biases(gpu, kind, dim, cap, bias, span, masks, kernel):
    Call(gpu, kind, ODD, 4, 4, dim, cap=cap, bias=bias, span=span, **masks).describe(kernel=kernel).run().check()


@pytest.mark.parametrize("kind,dim,lengths,heads", [("f16", 80, [300, 17, 257] + [5] * 60, 8), ("bf16", 96, [256] + [1] * 70, 8), ("bf16", 128, [4097, 300], 20)])
@pytest.mark.parametrize("cap,bias,span", [(0.0, None, 0), (9.0, "table", 30), (0.0, "slopes", 0)])
def test_tiles_of_256_queries(gpu, kind, dim, lengths, heads, cap, bias, span):
    """Sizes that take eight waves a workgroup: 512 and more tiles of 256 queries, of heads of 80 and 96, or of 4,096 queries."""
    c = Call(gpu, kind, lengths, heads, heads if dim < 128 else 1, dim, after=0, before=900, cap=cap, bias=bias, span=span, prefix=dim != 96)
    c.describe(kernel=_lib.ATTEND_MANY)
    assert (max(lengths) + 255) // 256 * len(lengths) * heads >= 512 or dim == 128
    c.run()
    if dim < 128:
        c.check()
        return
    torch().cuda.synchronize()  # two heads of the long ones against 64 bits
    got = c.out.double().cpu().numpy()
    q, kv = c.q.double().cpu().numpy(), c.kv.double().cpu().numpy()
    for h in (0, heads - 1):
        rows, keys = slice(c.q0[0], c.q0[0] + lengths[0]), slice(c.k0[0], c.k0[0] + lengths[0])
        want, bound = A.attend(q[rows, h:h + 1, :dim], kv[keys, :1, :dim], kv[keys, 1:, :dim], c.scale, c.cap,
                               None if c.slopes is None else c.slopes[h:h + 1], None if c.table is None else c.table[h:h + 1], 900, 0,
                               c.prefix[0], None, kind)
        assert (np.abs(got[rows, h:h + 1, :dim] - want) <= bound).all()


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (7, 1), (8, 2), (40, 1), (12, 12)])
@pytest.mark.parametrize("queries", [1, 2, 5])
@pytest.mark.parametrize("bias,span", [b[1:] for b in BIASES], ids=[b[0] for b in BIASES])
def test_single_tokens(gpu, heads, kv_heads, queries, bias, span):
    keys = [queries, queries + 1, 31, 32, 33, 129, 1000, 64]
    c = Call(gpu, "f16", [queries] * 8, heads, kv_heads, 64, key_lengths=keys, after=0, bias=bias, span=span, cap=11.0)
    for kernel in (_lib.ATTEND_PLANNED, _lib.ATTEND_FEW, _lib.ATTEND_MANY):
        c.out.fill_(9.0)
        c.describe(kernel=kernel).run().check()


@pytest.mark.parametrize("kind,dim", [("f16", 64), ("bf16", 80), ("bf16", 128), ("f16", 256), ("f16", 152)])
@pytest.mark.parametrize("masks", [dict(), dict(after=0), dict(after=0, before=3000), dict(after=0, before=700, prefix=True)],
                         ids=["all", "causal", "window", "prefix"])
@pytest.mark.parametrize("queries", [1, 7, 40])
def test_long_keys_shared_by_workgroups(gpu, kind, dim, masks, queries):
    c = Call(gpu, kind, [queries, queries, 1], 4, 2, dim, key_lengths=[9001, 4500, 70], bias="slopes", **masks)
    c.describe(kernel=_lib.ATTEND_FEW)
    if not masks or "before" not in masks or "prefix" in masks or masks["before"] > 1024:
        assert c.workspace is not None
    c.run().check()
    first = c.out.clone()
    c.out.fill_(9.0)
    c.run()
    torch().cuda.synchronize()
    assert torch().equal(first, c.out)  # equal calls, equal bits


@pytest.mark.parametrize("queries,keys,masks", [(300, 1000, dict(after=0)), (100, 40, dict(after=0)), (257, 513, dict(before=64, after=0)),
                                                (130, 0, dict()), (64, 2000, dict(after=3))])
@KERNELS
def test_queries_and_keys_of_different_lengths(gpu, queries, keys, masks, kernel):
    """Later pieces of prompts; more queries than keys (the first see nothing); no keys at all."""
    c = Call(gpu, "bf16", [queries] + [11] * 9, 8, 4, 64, key_lengths=[keys] + [23] * 9, bias="table", span=64, **masks)
    c.describe(kernel=kernel).run().check()


@pytest.mark.parametrize("span", [0, 1, 32, 500, 1024])
@KERNELS
def test_table_spans(gpu, span, kernel):
    Call(gpu, "f16", [700, 3, 130], 6, 6, 64, bias="table", span=span).describe(kernel=kernel).run().check()
    Call(gpu, "bf16", [700, 3, 130], 6, 3, 256, bias="table", span=span, cap=20.0, after=0).describe(kernel=kernel).run().check()


@pytest.mark.parametrize("cap", [1e-10, 0.01, 200.0, 1024.0])
@KERNELS
def test_smallest_and_largest_caps(gpu, cap, kernel):
    for kind, bias in (("f16", None), ("bf16", "slopes")):
        Call(gpu, kind, [300, 7], 4, 2, 64, bias=bias, cap=cap, after=0).describe(kernel=kernel).run().check()


@KERNELS
def test_rows_without_keys_are_zeros(gpu, kernel):
    c = Call(gpu, "f16", [200, 70], 4, 2, 64, documents=True)
    c.bounds[c.q0[0] + 10:c.q0[0] + 150] = [50, 50]
    c.bounds[c.q0[0] + 3] = [2 ** 31 - 1, -2 ** 31]
    c.bounds[c.q0[0] + 4] = [-5, 10 ** 9]  # cut to the keys
    c.describe(kernel=kernel).run().check()
    assert not c.out[c.q0[0] + 10:c.q0[0] + 150, :, :64].any()


@KERNELS
def test_biases_of_the_lowest_value_hide(gpu, kernel):
    c = Call(gpu, "bf16", [150, 90], 4, 4, 64, bias="table", span=100)
    c.table[:, :90] = np.finfo(np.float32).min
    c.table[1, 95:] = np.finfo(np.float32).min
    c.table[2, :] = -np.inf
    c.table[3, :] = np.finfo(np.float32).min  # a head that sees nothing
    c.describe(kernel=kernel).run().check()
    assert not c.out[c.q0[0]:c.q0[0] + 150, 2:, :64].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("cap", [0.0, 9.0])
@pytest.mark.parametrize("queries,keys", [([200, 90], [200, 90]), ([1, 3], [5000, 300])], ids=["prompt", "step"])
@KERNELS
def test_hidden_keys_may_hold_anything(gpu, bad, cap, queries, keys, kernel):
    """Not finite keys and values at places that some rows see and others do not: rows that do not see them are as if they were
    not there; rows that see a NaN are NaN."""
    c = Call(gpu, "f16", queries, 4, 2, 64, key_lengths=keys, after=0, before=60, cap=cap, bias="slopes")
    c.kv[c.k0[0] + keys[0] - 30, 2, 5] = bad       # a value that the last rows see (head 0 of v, dim 5)
    c.kv[c.k0[0] + keys[0] - 80, 1, 7] = bad       # keys behind some rows' windows
    c.kv[c.k0[0] + keys[0] - 90, 3, :64] = bad
    c.kv[c.k0[1]:c.k0[1] + 20, :, :64] = bad
    c.describe(kernel=kernel).run()
    torch().cuda.synchronize()
    got = c.out.double().cpu().numpy()
    want, bound = c.expected()
    # A row that sees an infinite score or value: infinite or no number in both, and which of them is the summation's matter.
    odd = ~np.isfinite(want)
    assert not np.isfinite(got[odd]).any()
    assert np.isfinite(got[~odd]).all()
    assert (np.abs(got[~odd] - want[~odd]) <= bound[~odd]).all()
    assert (~odd[c.q0[0]:c.q0[0] + queries[0]]).any()


def test_starts_and_lengths_are_cut_to_the_arrays(gpu):
    """Sequences that begin or end outside the arrays, or are longer than the call says: cut, and those that begin outside are none."""
    for kernel in (_lib.ATTEND_MANY, _lib.ATTEND_FEW):
        c = Call(gpu, "f16", [100, 50, 60, 70], 4, 2, 64, after=-1)
        c.describe(kernel=kernel)
        c.nq[3], c.nk[3] = 10 ** 9, 10 ** 9      # cut to max_q and max_k, and at the arrays' ends
        d = c.kept
        d["nq"].copy_(c.up(c.nq))
        d["nk"].copy_(c.up(c.nk))
        d["q0"][1] = -5
        d["k0"][2] = 10 ** 9
        c.run()
        torch().cuda.synchronize()
        got = c.out.clone()
        assert (got[c.q0[1]:c.q0[1] + 50] == 9).all()            # no queries
        assert not got[c.q0[2]:c.q0[2] + 60, :, :64].any()       # no keys: zeros
        rows = c.q.shape[0]
        c.nq[3], c.nk[3] = min(c.call.max_q, rows - c.q0[3]), min(c.call.max_k, c.kv.shape[0] - c.k0[3])
        # Rows past the sequence's own are now its queries and keys; here they hold NaNs, so its rows are NaN.
        if c.nk[3] > 70:
            assert got[c.q0[3]:c.q0[3] + 70, :, :64].isnan().all()


def test_a_cache_past_32_bits(gpu):
    """Rows 2^22 elements apart: the last lie more than 2^32 bytes behind the first."""
    t = torch()
    row, n, dim = 1 << 22, 1100, 64
    cache = t.empty(n * row, dtype=t.float16, device=gpu)
    kv = cache.as_strided((n, 2, dim), (row, dim, 1))
    gen = t.Generator(device=gpu).manual_seed(3)
    kv.copy_(t.randn(n, 2, dim, generator=gen, device=gpu))
    for queries, n_seq in ((1, 1), (300, 100)):
        c = Call(gpu, "f16", [queries] * n_seq, 4, 1, dim, key_lengths=[n] * n_seq, after=0)
        c.kv = kv
        c.k0 = np.zeros(n_seq, np.int32)
        c.describe(k_row=row, v_row=row, k_head=dim, v_head=dim, k_rows=n, v=kv.data_ptr() + 2 * dim)
        c.run()
        t.cuda.synchronize()
        got = c.out.double().cpu().numpy()
        want, bound = A.attend(c.q[c.q0[0]:c.q0[0] + queries, :, :dim].double().cpu().numpy(), kv[:, :1].double().cpu().numpy(),
                               kv[:, 1:].double().cpu().numpy(), c.scale, after=0, kind="f16")
        assert (np.abs(got[c.q0[0]:c.q0[0] + queries, :, :dim] - want) <= bound).all()


def test_no_keys_at_all(gpu):
    """An empty cache: no pointers, zeros."""
    for kernel in (_lib.ATTEND_PLANNED, _lib.ATTEND_MANY, _lib.ATTEND_FEW):
        c = Call(gpu, "f16", [40, 1], 4, 2, 64, key_lengths=[0, 0])
        c.describe(k=None, v=None, k_rows=0, max_k=0, kernel=kernel).run().check()
        assert not c.out[c.q0[0]:c.q0[0] + 40, :, :64].any()


def test_head_major_planes(gpu):
    """The strides of [heads][rows][dim]."""
    t = torch()
    c = Call(gpu, "bf16", [90, 40], 4, 2, 64, after=0)
    q, kv, out = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (c.q, c.kv, c.out))
    c.describe(q=at(q), k=at(kv), v=kv.data_ptr() + 2 * 2 * kv.stride(1), out=at(out), q_row=q.stride(0), q_head=q.stride(1),
               k_row=kv.stride(0), k_head=kv.stride(1), v_row=kv.stride(0), v_head=kv.stride(1), out_row=out.stride(0), out_head=out.stride(1))
    c.run()
    c.out = out
    c.check()
    assert t.is_tensor(out)


@pytest.mark.parametrize("queries", [1, 200])
def test_graphs_with_lengths_that_change_and_workspaces_of_their_own(gpu, queries):
    t = torch()
    n = 3 if queries == 1 else 40
    c = Call(gpu, "f16", [queries] * n, 8, 8, 64, key_lengths=[6000 if queries == 1 else 400] * n, after=0, bias="slopes").describe()
    d = Call(gpu, "f16", [queries] * n, 8, 8, 64, key_lengths=[6000 if queries == 1 else 400] * n, after=0, cap=5.0, seed=5).describe()
    t.cuda.synchronize()
    side = t.cuda.Stream()
    c.run(side)
    side.synchronize()
    c.check()
    graphs = []
    for x in (c, d):
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g):
            x.run()
        graphs.append(g)
    for keys in (300, 6000, 1, 2500):
        for x, g in zip((c, d), graphs):
            x.nk = np.minimum(np.array([keys, 300 + queries, queries] + [queries + 30] * n, np.int32)[:n], x.call.max_k)
            x.kept["nk"].copy_(x.up(x.nk))
            x.out.fill_(9.0)
        t.cuda.synchronize()
        for g in graphs:
            g.replay()
        t.cuda.synchronize()
        for x in (c, d):
            x.check()


# ---------------- document bounds ----------------

@pytest.mark.parametrize("mean", [1, 3, 70, 900, 10 ** 9])
def test_document_bounds(gpu, mean):
    t, lib = torch(), _lib.load()
    rng = np.random.default_rng(mean)
    lengths = np.array([1, 0, 64, 65, 5000, 63, 128, 2049], np.int32)
    starts = (np.cumsum(lengths + 2) - lengths).astype(np.int32)
    rows = int(starts[-1] + lengths[-1] + 2)
    ids = np.full(rows, 7, np.int32)
    want = np.full((rows, 2), -9, np.int32)
    for s, n in zip(starts, lengths):
        ids[s:s + n] = rng.integers(-3, 3) + np.cumsum(rng.random(n) < 1 / mean) % 5  # ids come again
        want[s:s + n] = A.document_bounds(ids[s:s + n])
    got = t.full((rows, 2), -9, dtype=t.int32, device=gpu)
    d, s, n = (t.from_numpy(x).to(gpu) for x in (ids, starts, lengths))
    _lib.check(lib.laya_op_document_bounds(at(d), at(s), at(n), len(lengths), rows, 5000, at(got), None))
    t.cuda.synchronize()
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    got.fill_(-9)
    _lib.check(lib.laya_op_document_bounds(at(d), at(s), at(n), len(lengths), rows, 100, at(got), None))  # longer ones are cut
    t.cuda.synchronize()
    for a, m in zip(starts, np.minimum(lengths, 100)):
        np.testing.assert_array_equal(got.cpu().numpy()[a:a + m], A.document_bounds(ids[a:a + m]))
        assert (got.cpu().numpy()[a + m:a + m + 2] == -9).all()


# ---------------- together ----------------

@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_projection_rotary_and_attention_together(gpu, kind):
    """A layer's attention as a caller builds it: the packed projection, both halves turned in place, documents found, attention over
    the rows where they lie, against each step in 64 bits; and, without documents, against laya_op_qkv with laya_op_attention."""
    t, lib = torch(), _lib.load()
    rng = np.random.default_rng(4)
    dtype = {"f16": t.float16, "bf16": t.bfloat16}[kind]
    heads, dim, lengths = 4, 64, [96, 160, 48]
    width, m = heads * dim, sum(lengths)
    starts = np.cumsum(lengths) - lengths
    x = t.from_numpy(rng.normal(0, 1, (m, width))).to(gpu).to(dtype)
    w = t.from_numpy(rng.normal(0, width ** -0.5, (3 * width, width))).to(gpu).to(dtype)
    positions = np.concatenate([np.arange(n) for n in lengths]).astype(np.int32)
    turns = (ct.c_double * 32)()
    _lib.check(lib.laya_rotary_frequencies(_lib.FREQ_PLAIN, 10000.0, 64, 1.0, 0.0, 0.0, 0.0, turns))
    turns = np.array(turns)
    stream = ct.c_void_p(t.cuda.current_stream().cuda_stream)
    up = lambda a: t.from_numpy(np.ascontiguousarray(a)).to(gpu)  # noqa: E731
    packed = t.empty(m, 3 * heads, dim, dtype=dtype, device=gpu)
    _lib.check(lib.laya_op_linear(at(x), at(w), None, at(packed), 1, CODE[kind], m, 3 * width, width, 1, -1, stream))
    before = packed.double().cpu().numpy()
    p, f = up(positions), up(turns)
    _lib.check(lib.laya_op_rotary(at(packed), 3 * width, dim, at(packed), 3 * width, dim, CODE[kind], at(p), at(f), 1.0, 0, 1, m, 2 * heads,
                                  dim, dim, stream))
    turned = packed.double().cpu().numpy()
    want = A.rotate(before[:, :2 * heads], positions, turns)
    assert (np.abs(turned[:, :2 * heads] - want) <= A.HALF[kind] * np.abs(want) + 1e-6 * np.abs(before[:, :2 * heads]).max()).all()
    np.testing.assert_array_equal(turned[:, 2 * heads:], before[:, 2 * heads:])
    ids = np.concatenate([np.cumsum(rng.random(n) < .05) for n in lengths]).astype(np.int32)
    documents, s0, n0, bounds = up(ids), up(starts.astype(np.int32)), up(np.array(lengths, np.int32)), t.full((m, 2), -1, dtype=t.int32, device=gpu)
    _lib.check(lib.laya_op_document_bounds(at(documents), at(s0), at(n0), 3, m, max(lengths), at(bounds), stream))
    out = t.empty(m, heads, dim, dtype=dtype, device=gpu)
    call = _lib.LayaAttend(struct_bytes=ct.sizeof(_lib.LayaAttend), dtype=CODE[kind], q=at(packed), k=packed.data_ptr() + 2 * width,
                           v=packed.data_ptr() + 4 * width, out=at(out), q_row=3 * width, q_head=dim, k_row=3 * width, k_head=dim,
                           v_row=3 * width, v_head=dim, out_row=width, out_head=dim, heads=heads, kv_heads=heads, dim=dim, q_rows=m,
                           k_rows=m, n_seq=3, max_q=max(lengths), max_k=max(lengths), q_starts=at(s0), q_lengths=at(n0), k_starts=at(s0),
                           k_lengths=at(n0), scale=0.125, before=-1, after=-1, bounds=at(bounds))
    assert lib.laya_attend_workspace(ct.byref(call)) == 0

    def compare(bounded):
        _lib.check(lib.laya_op_attend(ct.byref(call), None, 0, stream))
        got = out.double().cpu().numpy()
        for a, n in zip(starts, lengths):
            rows = slice(a, a + n)
            b = A.document_bounds(ids[rows]) if bounded else None
            want, bound = A.attend(turned[rows, :heads], turned[rows, heads:2 * heads], turned[rows, 2 * heads:], 0.125, bounds=b, kind=kind)
            assert (np.abs(got[rows] - want) <= bound).all()
        return got

    compare(True)
    call.bounds = None
    got = compare(False)

    # The fused projection and its attention: the same roundings in another order, each within its bound of the same values.
    cos, sin = (up(fn(2 * np.pi * np.arange(max(lengths))[:, None] * turns).astype(np.float32)) for fn in (np.cos, np.sin))
    q, k, vt = (t.empty(heads * m * dim, dtype=dtype, device=gpu) for _ in range(3))
    _lib.check(lib.laya_op_qkv(at(x), at(w), None, at(q), at(k), at(vt), at(cos), at(sin), at(p), CODE[kind], m, width, -1, stream))
    tiles = np.zeros((m // 16, 4), np.int32)
    ip = ct.POINTER(ct.c_int32)
    block = lib.laya_attention_block(1, 4)
    a32, l32 = starts.astype(np.int32), np.array(lengths, np.int32)
    used = lib.laya_attention_tiles(a32.ctypes.data_as(ip), l32.ctypes.data_as(ip), 3, m, block, tiles.ctypes.data_as(ip), m // 16)
    assert used > 0
    listed, fused = up(tiles), t.empty(m, heads, dim, dtype=dtype, device=gpu)
    _lib.check(lib.laya_op_attention(at(q), at(k), at(vt), at(fused), at(listed), m, heads, m // 16, 1, 4, -1, CODE[kind], stream))
    t.cuda.synchronize()
    # Its rotation rounds once where the other path rounds the projection and the rotation: scores differ by two roundings of
    # queries and keys, 4 h of the sum of |q||k|, and the weights by as much.
    for a, n in zip(starts, lengths):
        rows = slice(a, a + n)
        _, bound = A.attend(turned[rows, :heads], turned[rows, heads:2 * heads], turned[rows, 2 * heads:], 0.125, kind=kind)
        score = 0.125 * np.linalg.norm(turned[rows, :heads], axis=-1).max() * np.linalg.norm(turned[rows, heads:2 * heads], axis=-1).max()
        largest = np.abs(turned[rows, 2 * heads:]).max()
        allowed = 2 * bound + (2 * 4 * A.HALF[kind] * score + A.HALF[kind]) * largest
        assert (np.abs(got[rows] - fused.double().cpu().numpy()[rows]) <= allowed).all()
