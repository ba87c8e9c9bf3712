"""Building the op module leaves the environment as it was, and takes the compiler that the caller names."""
import os
import shutil

import pytest
import torch.utils.cpp_extension

from flashgmm_b200 import build


@pytest.mark.parametrize("before", [None, "/opt/other/bin/g++"])
@pytest.mark.parametrize("named", [None, "/opt/mine/bin/g++"])
@pytest.mark.parametrize("fails", [False, True])
def test_compiler_and_environment(monkeypatch, before, named, fails):
    for name, value in (("CXX", before), ("FLASHGMM_CXX", named)):
        monkeypatch.delenv(name, raising=False) if value is None else monkeypatch.setenv(name, value)
    used = []

    def load(**kwargs):
        used.append(os.environ.get("CXX"))
        if fails:
            raise RuntimeError("does not compile")

    monkeypatch.setattr(torch.utils.cpp_extension, "load", load)
    monkeypatch.setattr(shutil, "copyfile", lambda *a: None)
    environment = dict(os.environ)
    if fails:
        with pytest.raises(RuntimeError, match="does not compile"):
            build.build_torch_ext()
    else:
        build.build_torch_ext()
    assert dict(os.environ) == environment
    assert used == [named or ("/usr/bin/g++" if os.path.exists("/usr/bin/g++") else before)]
