"""CPU tests of the grouped-head attention's C entries: NULL arguments are
refused with a message, nothing is launched."""
from __future__ import annotations

import ctypes as C


def test_null_arguments_are_refused():
    from wave_engine_b200 import _lib
    l = _lib.lib()
    d, c = _lib.GqaAttnDesc(), _lib.GqaCacheDesc()
    assert l.wb_gqa_attention(None, None) == _lib.WB_EINVAL
    assert l.wb_gqa_attention(None, C.byref(d)) == _lib.WB_EINVAL
    for cache in (None, C.byref(c)):
        assert l.wb_gqa_cache_write(None, cache, None, 1, None, 1, None, None, 0, 0, None, 0, 0) == _lib.WB_EINVAL
        assert l.wb_gqa_cache_read(None, cache, None, 1, None, 1, None, None, None) == _lib.WB_EINVAL
        assert l.wb_gqa_decode(None, cache, None, 1, 1, None, 0, 0, 1.0, None, None) == _lib.WB_EINVAL
    assert b"NULL" in l.wb_last_error()


def test_descriptors_match_the_header():
    """Field names and order of the ctypes descriptors are the header's."""
    import re
    from tests.conftest import ROOT
    from wave_engine_b200 import _lib
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "wave_b200.h").read_text(), flags=re.S)
    for name, cls in (("wb_gqa_attn_desc", _lib.GqaAttnDesc), ("wb_gqa_cache_desc", _lib.GqaCacheDesc)):
        body = text[:text.index("} " + name)].rsplit("typedef struct {", 1)[1]
        want = []
        for line in body.split(";"):
            m = re.match(r"\s*(?:const\s+)?(int32_t|int64_t|float|void)\s+(.*)", line.strip(), re.S)
            if m:
                for f in m.group(2).split(","):
                    f = f.strip()
                    want.append((f.lstrip("*"), "p" if f.startswith("*") else m.group(1)))
        kind = {C.c_int32: "int32_t", C.c_int64: "int64_t", C.c_float: "float", C.c_void_p: "p"}
        assert [(n, kind[t]) for n, t in cls._fields_] == want


def test_packed_descriptors_are_the_ctypes_ones():
    """The struct formats that the entry points pack with lay every field where the descriptors have it."""
    from wave_engine_b200 import _lib, gqa
    for fmt, cls in ((gqa._ATTN, _lib.GqaAttnDesc), (gqa._CACHE, _lib.GqaCacheDesc)):
        assert fmt.size == C.sizeof(cls)
        values = [i + 1 for i in range(len(cls._fields_))]
        d = cls.from_buffer_copy(fmt.pack(*values))
        assert [getattr(d, n) for n, _ in cls._fields_] == values
