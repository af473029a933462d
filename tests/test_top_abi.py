"""The entry points on the top of a row of logits: descriptors as the header has them, bad ones refused on the host."""
import re

import pytest

from test_lib_abi import HEADER


def test_packed_descriptors_match_the_header():
    from sparseforge_amd import _lib as L

    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    for name, fmt in (("sf_sample_desc", L.SAMPLE_DESC), ("sf_top_logits_desc", L.TOP_LOGITS_DESC),
                      ("sf_top_kl_desc", L.TOP_KL_DESC)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        got = ""
        for field in filter(None, (f.strip() for f in body.split(";"))):
            code = "q" if "*" in field or field.startswith("int64_t") else {"int": "i", "float": "f"}[field.split()[0]]
            got += code * (field.count(",") + 1)
        want = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qif])", fmt.format))
        assert got == want, name


SOME = 1 << 20  # an address that nothing reads: every call here is refused before a launch


def test_sampling_refuses_bad_descriptors():
    from sparseforge_amd import _lib as L

    lib = L.load()

    def call(x=SOME, stride=8, rows=2, vocab=8, u=SOME, tokens=SOME, temperature=1.0, dtype=L.DT_F32):
        return lib.sf_sample_logits(L.SAMPLE_DESC.pack(x, stride, rows, vocab, u, tokens, 0, 0, 0, 0, 0, temperature, 1.0,
                                                       0.0, 0, dtype), None)

    for bad in ({"dtype": 2}, {"rows": -1}, {"vocab": 0}, {"vocab": 262145}, {"x": 0}, {"u": 0}, {"tokens": 0},
                {"stride": -1}, {"temperature": -1.0}, {"temperature": float("nan")}, {"rows": 1 << 31}):
        assert call(**bad) == L.SF_ERR_INVALID, bad
        assert "sf_sample_logits" in L.last_error()
    assert call(rows=0) == L.SF_OK
    assert lib.sf_sample_logits(None, None) == L.SF_ERR_INVALID


def test_top_logits_refuses_bad_descriptors():
    from sparseforge_amd import _lib as L

    lib = L.load()

    def call(x=SOME, outer=0, step=8, inner=2, rows=2, vocab=2000, k=3, values=SOME, ids=SOME, T=1.0, dtype=L.DT_F32):
        return lib.sf_top_logits(L.TOP_LOGITS_DESC.pack(x, outer, step, inner, rows, vocab, k, values, ids, 0, T, dtype),
                                 None)

    for bad in ({"dtype": 2}, {"rows": -1}, {"vocab": 0}, {"vocab": 262145}, {"k": 0}, {"k": 1025}, {"vocab": 2, "k": 3},
                {"inner": 0}, {"inner": 3}, {"outer": -1}, {"step": -1}, {"x": 0}, {"values": 0}, {"ids": 0}, {"T": 0.0},
                {"T": float("inf")}, {"T": float("nan")}):
        assert call(**bad) == L.SF_ERR_INVALID, bad
        assert "sf_top_logits" in L.last_error()
    assert call(rows=0) == L.SF_OK
    assert lib.sf_top_logits(None, None) == L.SF_ERR_INVALID


@pytest.mark.parametrize("entry", ["forward", "backward", "double_backward"])
def test_top_kl_refuses_bad_descriptors(entry):
    from sparseforge_amd import _lib as L

    lib = L.load()

    def call(s=SOME, outer=0, step=8, inner=2, rows=2, vocab=50, values=SOME, ids=SOME, k=3, stats=SOME, norm=SOME, T=1.0,
             dtype=L.DT_F32, vdt=L.DT_F32, id_bytes=4, ws=SOME, size=1 << 20, out=SOME):
        d = L.TOP_KL_DESC.pack(s, outer, step, inner, rows, vocab, values, ids, k, 0, 0, stats, norm, T, dtype, vdt,
                               id_bytes)
        if entry == "forward":
            return lib.sf_top_kl_forward(d, out, ws, size, None)
        if entry == "backward":
            return lib.sf_top_kl_backward(d, SOME, out, None)
        return lib.sf_top_kl_double_backward(d, SOME, SOME, out, None, ws, size, None)

    bads = [{"dtype": 2}, {"vdt": 2}, {"rows": 0}, {"vocab": 0}, {"vocab": 262145}, {"inner": 0}, {"inner": 3},
            {"outer": -1}, {"step": -1}, {"k": -1}, {"k": 51}, {"id_bytes": 2}, {"s": 0}, {"values": 0}, {"ids": 0},
            {"stats": 0}, {"norm": 0}, {"T": 0.0}, {"T": float("nan")}, {"T": float("inf")}, {"out": 0}]
    if entry != "backward":
        bads += [{"ws": 0}, {"size": 8}]
    for bad in bads:
        assert call(**bad) == L.SF_ERR_INVALID, bad
        assert "sf_top_kl_" + entry in L.last_error()
    assert lib.sf_top_kl_stats_size(0) == 0 and lib.sf_top_kl_workspace_size(0) == 0


def test_rows_of_a_view():
    """How the binding describes rows: two strides at most, others copied."""
    import torch

    from sparseforge_amd import _lib as L

    x = torch.arange(2 * 5 * 3 * 7).view(2, 5, 3, 7)
    for t in (x, x[:, :-1], x[:, :, 0], x[0, 0, 0], x[:, ::2, 1:], x.transpose(0, 1), x.transpose(-1, -2), x[:, :1],
              x[..., 2:5], x[:1].expand(4, 5, 3, 7), x[0, 0, 0, :1].expand(3, 1)):
        y, outer, step, inner, rows = L.rows_of(t)
        assert y.shape == t.shape and rows == t.shape[:-1].numel() and rows % inner == 0
        flat = torch.as_strided(y, (rows // inner, inner, t.shape[-1]), (outer, step, 1), y.storage_offset())
        assert torch.equal(flat.reshape(t.shape), t)
    assert L.rows_of(x[:, :-1])[0].data_ptr() == x.data_ptr() and L.rows_of(x[:0])[4] == 0


def test_limits_of_temperatures_and_entries():
    """Temperatures whose reciprocal float32 does not hold, and lists that are too long, are refused."""
    from sparseforge_amd import _lib as L

    lib = L.load()
    for T in (1e-39, 1e-31, 1e31, 3.4e38):
        d = L.TOP_LOGITS_DESC.pack(SOME, 0, 8, 2, 2, 2000, 3, SOME, SOME, 0, T, L.DT_F32)
        assert lib.sf_top_logits(d, None) == L.SF_ERR_INVALID
    for T, k in ((1e-39, 3), (3.4e38, 3), (1.0, 4097)):
        d = L.TOP_KL_DESC.pack(SOME, 0, 8, 2, 2, 50000, SOME, SOME, k, 0, 0, SOME, SOME, T, L.DT_F32, L.DT_F32, 4)
        assert lib.sf_top_kl_forward(d, SOME, SOME, 1 << 20, None) == L.SF_ERR_INVALID
        assert lib.sf_top_kl_backward(d, SOME, SOME, None) == L.SF_ERR_INVALID
        assert lib.sf_top_kl_double_backward(d, SOME, SOME, SOME, None, SOME, 1 << 20, None) == L.SF_ERR_INVALID
