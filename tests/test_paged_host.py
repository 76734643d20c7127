"""The paged cache's host side without a GPU: refusals that happen before any device is needed."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")


def test_null_contexts_are_refused_not_followed():
    from maryml_b200 import _lib
    lib = _lib.lib
    kv, terms = _lib.PagedKv(), _lib.ScoreTerms()
    assert lib.mb_paged_append(None, None, None, 0, 0, 0, C.byref(kv), None, None, None, 0, None, None) == _lib.ERR_INVALID
    assert lib.mb_paged_append(None, None, None, 0, 0, 0, None, None, None, None, 0, None, None) == _lib.ERR_INVALID
    assert lib.mb_paged_decode(None, None, None, 1, 1, C.byref(kv), C.byref(terms), None, None, 0) == _lib.ERR_INVALID
    assert lib.mb_paged_prompt(None, None, None, 1, 1, C.byref(kv), None, C.byref(terms), None, None, 0) == _lib.ERR_INVALID
    assert lib.mb_paged_decode_workspace(None, C.byref(kv), 1, 1) == 0
    assert lib.mb_paged_prompt_workspace(None, C.byref(kv), 1, 1) == 0


def test_the_structures_match_the_header():
    """Field by field in the header's order: an ABI that drifted would read wild pointers."""
    import os
    import re
    from maryml_b200 import _lib
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mary_b200.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, cls in (("mb_paged_kv", _lib.PagedKv), ("mb_score_terms", _lib.ScoreTerms)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        fields = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            kind = C.c_void_p if "*" in decl else C.c_size_t if decl.startswith("size_t") else C.c_float if decl.startswith("float") else C.c_int
            fields += [(n.strip().split("*")[-1].split()[-1], kind) for n in decl.split(",")]
        assert fields == [(n, t) for n, t in cls._fields_]


def test_pools_on_the_host_are_refused():
    from maryml_b200 import MaryError
    from maryml_b200.paged import PagedCache
    k = torch.zeros((4, 16, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(MaryError):
        PagedCache(k, k)
    codes, scales = torch.zeros((4, 16, 128), dtype=torch.uint8), torch.zeros((4, 16, 16), dtype=torch.uint8)
    with pytest.raises(MaryError):
        PagedCache(codes, codes, scales, scales, head_dim=128)
