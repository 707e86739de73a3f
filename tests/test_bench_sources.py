"""The sources that bench.py hashes are those that the headline kernel is compiled from."""
import hashlib
import os
import re

import bench


def test_every_included_file_is_hashed():
    csrc = os.path.dirname(bench.KERNEL_SOURCES[0])
    found, todo = [], ["attn.hip"]
    while todo:
        name = todo.pop(0)
        path = os.path.join(csrc, name)
        if name in found or not os.path.exists(path):  # the public header is no part of the kernels
            continue
        found.append(name)
        todo += re.findall(r'#include "([^"]+)"', open(path).read())
    assert [os.path.basename(p) for p in bench.KERNEL_SOURCES] == found


def test_a_change_in_any_of_them_shows(tmp_path, monkeypatch):
    now = bench.kernel_source_sha256()
    text = b"".join(open(p, "rb").read() for p in bench.KERNEL_SOURCES)
    assert now == hashlib.sha256(text).hexdigest()[:16]
    for i, p in enumerate(bench.KERNEL_SOURCES):
        changed = tmp_path / os.path.basename(p)
        changed.write_bytes(open(p, "rb").read() + b"\n")
        monkeypatch.setattr(bench, "KERNEL_SOURCES", [str(changed) if j == i else q
                                                      for j, q in enumerate(bench.KERNEL_SOURCES)])
        assert bench.kernel_source_sha256() != now
        monkeypatch.undo()
