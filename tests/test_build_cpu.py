"""What building the kernel library needs."""
from kernelcodegen_b200 import build


def test_the_kernel_library_builds_without_torch(native_lib, monkeypatch):
    """nvcc (and g++ for the C++ operator API) is enough: the C-ABI's users need neither torch nor its binding."""
    def never(*a, **k):
        raise AssertionError("the torch binding was built")

    monkeypatch.setattr(build, "build_binding", never)
    assert build.build() == build.LIB_PATH
    assert build.build_host() == build.HOST_LIB_PATH
