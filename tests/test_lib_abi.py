"""The C-ABI library: every function include/sparseforge_amd.h declares is exported
and bound, and the device tie table equals the torch.topk fixture (CPU only)."""
import json
import os
import re

import pytest

from conftest import GOLDEN, REPO

HEADER = os.path.join(REPO, "include", "sparseforge_amd.h")


def header_functions():
    text = open(HEADER).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(sf_\w+)\s*\(", text, flags=re.M)))


def test_header_declares_entry_points():
    names = header_functions()
    assert "sf_gemm" in names and "sf_update_mask" in names and len(names) >= 10


def test_library_exports_every_declared_symbol():
    from sparseforge_amd import _lib as L

    if not os.path.exists(L.LIB_PATH):
        pytest.fail(f"HIP library not built at {L.LIB_PATH}")
    lib = L.load()
    names = header_functions()
    missing = [n for n in names if not hasattr(lib, n)]
    assert not missing, missing
    assert sorted(L.SIGNATURES) == names, "ctypes bindings differ from the header"
    assert lib.sf_version() >= 100


def test_error_path_without_gpu():
    """An invalid call is rejected on the host before any device work."""
    from sparseforge_amd import _lib as L

    lib = L.load()
    rc = lib.sf_hard_mask(None, 7, None, 0, 4, 4, 2, 2, 4, None)
    assert rc == L.SF_ERR_INVALID
    assert "dtype" in L.last_error()
    d = L.GemmDesc()
    d.dtype = 5
    assert lib.sf_gemm(L.byref(d), None) == L.SF_ERR_INVALID


def test_device_tie_table_matches_fixture():
    src = open(os.path.join(REPO, "sparseforge_amd", "csrc", "sf_common.hpp")).read()
    body = src[src.index("kTopkTies4[3][256] = {"):]
    body = body[: body.index("};")]
    rows = re.findall(r"\{([\d,\s]+)\}", body.split("=", 1)[1])
    tables = [[int(v) for v in r.replace("\n", "").split(",") if v.strip()] for r in rows]
    fx = json.load(open(os.path.join(GOLDEN, "topk_ties_m4.json")))["tables"]
    for k in (1, 2, 3):
        expect = [0] * 256
        for key, row in fx[str(k)].items():
            expect[int(key)] = row["keep"]
        assert tables[k - 1] == expect, f"k={k}"


def test_product_package_never_uses_the_oracle_or_scratch_files():
    """The product path (sparseforge_amd/) imports nothing from oracle/ (test infrastructure) and
    reads nothing under _work/ (the builder's scratch space)."""
    import ast
    import pathlib

    pkg = pathlib.Path(__file__).resolve().parents[1] / "sparseforge_amd"
    for path in pkg.rglob("*.py"):
        tree = ast.parse(path.read_text())
        for node in ast.walk(tree):
            if isinstance(node, ast.Import):
                names = [a.name for a in node.names]
            elif isinstance(node, ast.ImportFrom):
                names = [node.module or ""]
            else:
                continue
            assert not any(n == "oracle" or n.startswith("oracle.") for n in names), f"{path} imports the oracle"
        assert "_work/" not in path.read_text(), f"{path} refers to _work/"
    for path in list(pkg.rglob("*.hip")) + list(pkg.rglob("*.hpp")):
        assert "_work/" not in path.read_text(), f"{path} refers to _work/"


def test_packed_descriptors_match_the_header():
    """sf_rotary_desc and sf_logits_desc field by field against the struct formats that the binding packs."""
    from sparseforge_amd import _lib as L

    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    for name, fmt in (("sf_rotary_desc", L.ROTARY_DESC), ("sf_logits_desc", L.LOGITS_DESC)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        got = ""
        for field in filter(None, (f.strip() for f in body.split(";"))):
            code = "q" if "*" in field or field.startswith("int64_t") else {"int": "i", "float": "f"}[field.split()[0]]
            got += code * (field.count(",") + 1)
        want = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qif])", fmt.format))
        assert got == want, name


def test_generation_entry_points_refuse_on_the_host():
    """Bad descriptors of the operators for generation come back as errors before any device work."""
    from sparseforge_amd import _lib as L

    lib = L.load()
    some = 1 << 12  # an address that is looked at only once the rest is right
    assert lib.sf_rotary(None, None) == L.SF_ERR_INVALID and lib.sf_process_logits(None, None) == L.SF_ERR_INVALID

    def rotary(D=64, r=64, S=4, rows=8, dtype=1, q=some, pos=0, pos_bytes=0, B=1, H=2):
        return lib.sf_rotary(L.ROTARY_DESC.pack(q, some, 0, 0, 0, H, 0, 0, 0, 0, 0, 0, B, S, D, r, some, some, rows, pos,
                                                0, pos_bytes, dtype, 0, 0), None)

    for bad in (dict(r=63), dict(r=66), dict(r=0), dict(D=0), dict(D=5000, r=2), dict(rows=3), dict(dtype=2),
                dict(q=0), dict(pos=some, pos_bytes=2), dict(B=-1), dict(B=1 << 20, S=1 << 20), dict(H=1 << 21)):
        assert rotary(**bad) == L.SF_ERR_INVALID, bad
        assert "sf_rotary" in L.last_error()
    assert rotary(S=0) == L.SF_OK and rotary(B=0) == L.SF_OK and rotary(H=0) == L.SF_OK

    def logits(rows=2, vocab=9, dtype=0, x=some, stride=9, hist=0, hist_bytes=0, rep=1.0):
        return lib.sf_process_logits(L.LOGITS_DESC.pack(x, some, 9, stride, rows, vocab, hist, 3, 3, 0, 0, 0, 0, 0, 0, 0,
                                                        0, rep, 0.0, 0.0, hist_bytes, 0, dtype), None)

    for bad in (dict(rows=65536), dict(rows=-1), dict(vocab=1 << 31), dict(dtype=3), dict(x=0), dict(stride=8),
                dict(hist=some, hist_bytes=1), dict(rep=0.0)):
        assert logits(**bad) == L.SF_ERR_INVALID, bad
    assert logits(rows=0) == L.SF_OK and logits(vocab=0) == L.SF_OK

    def cache(**kw):
        d = L.Kv8Cache()
        for name, _ in L.Kv8Cache._fields_[:8]:
            setattr(d, name, some)
        d.batch, d.kv_heads, d.head_dim, d.blocks = 2, 2, 64, 4
        for name, value in kw.items():
            setattr(d, name, value)
        return L.byref(d)

    for bad in (dict(k_codes=0), dict(ends=0), dict(batch=0), dict(kv_heads=65536), dict(head_dim=60),
                dict(head_dim=264), dict(blocks=0), dict(v_tail=some + 2)):
        assert lib.sf_kv8_extend(cache(**bad), 1, None, None) == L.SF_ERR_INVALID, bad
    good = cache()
    assert lib.sf_kv8_extend(good, 257, None, None) == L.SF_ERR_INVALID
    for args in ((some + 2, 64, 64, 64, some, 64, 64, 64, 1), (some, 64, 60, 64, some, 64, 64, 64, 1),
                 (None, 64, 64, 64, some, 64, 64, 64, 1), (some, 64, 64, 64, some, 64, 64, 64, 257)):
        assert lib.sf_kv8_append(good, *args, None) == L.SF_ERR_INVALID, args
    assert lib.sf_kv8_append(good, None, 0, 0, 0, None, 0, 0, 0, 0, None) == L.SF_OK
    assert lib.sf_kv8_values(good, None, 0, 257, some, some, None) == L.SF_ERR_INVALID
    assert lib.sf_kv8_values(good, None, 0, 0, None, None, None) == L.SF_OK

    def attend(q=some, ss=64, n=1, heads=4, scale=1.0, window=0, bound=10, ws=0, size=0):
        return lib.sf_kv8_attend(good, q, 64, ss, 64, n, heads, scale, window, bound, some, ws, size, None)

    for bad in (dict(q=some + 2), dict(q=None), dict(ss=4), dict(n=257), dict(heads=3), dict(heads=1), dict(scale=0.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(bound=257), dict(bound=-1)):
        assert attend(**bad) == L.SF_ERR_INVALID, bad
    # keys in several pieces need a workspace
    big = cache(blocks=1024)
    size = lib.sf_kv8_attend_workspace_size(2, 2, 4, 64, 1, 60000)
    assert size > 0
    for ws, n in ((None, 0), (some, size - 1), (some + 4, size)):
        assert lib.sf_kv8_attend(big, some, 64, 64, 64, 1, 4, 1.0, 0, 60000, some, ws, n, None) == L.SF_ERR_INVALID
