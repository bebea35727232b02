"""The extension's build."""
import os

from runbookai_amd.ops import build as ext_build


def test_build_keeps_no_object_of_an_earlier_build(tmp_path, monkeypatch):
    import torch.utils.cpp_extension

    for fn in ("packed_attn_hip.cuda.o", ext_build.EXT_NAME + ".so", "build.ninja"):
        (tmp_path / fn).write_text("old")
    seen = []
    monkeypatch.setattr(ext_build, "BUILD_DIR", str(tmp_path))
    monkeypatch.setattr(torch.utils.cpp_extension, "load",
                        lambda **kw: seen.append(sorted(os.listdir(kw["build_directory"]))))
    ext_build.build()
    assert seen == [["build.ninja"]]
