"""No kernel of the rotary positions or the cross attention spills to scratch
(the compiler's own resource remarks on the committed sources)."""

import os
import re
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_kernel_resources import HIPCC, _remarks

FILES = ["rotary", "cross_fwd", "cross_bwd"]
pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")


def test_no_kernel_spills(tmp_path):
    with ThreadPoolExecutor(max_workers=len(FILES)) as ex:
        logs = list(ex.map(lambda f: _remarks(f, str(tmp_path)), FILES))
    found = {}
    for log in logs:
        name = None
        for line in log.splitlines():
            m = re.search(r"remark: Function Name: (\S+)", line)
            name = m.group(1) if m else name
            m = re.search(r"remark:\s+ScratchSize \[bytes/lane\]: (\d+)", line)
            if m and name:
                found[name] = int(m.group(1))
    for kind in ("rotary_table_kernel", "rotary_kernel", "cross_fwd_kernel", "cross_join_kernel",
                 "cross_words_kernel", "cross_dq_kernel", "cross_dkv_kernel", "cross_sum_kernel"):
        assert any(kind in n for n in found), kind
    assert not {n: s for n, s in found.items() if s}
