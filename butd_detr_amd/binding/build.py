"""Builds the ATen / pybind11 front ends of the C ABI in-tree with torch.utils.cpp_extension:

    python -m butd_detr_amd.binding.build   ->  butd_detr_amd/binding/_build/butd_pointnet2_aten.so
                                                butd_detr_amd/binding/_build/blocks/butd_blocks_aten.so

Plain C++ (no device code): they link libbutd_detr_hip.so (``python -m butd_detr_amd.build``) and torch.

* ``pointnet2_aten.cpp`` is the reference's module surface (``pointnet2._ext``, bindings.cpp:11-24).  The product path does
  not need it (it binds the same C ABI with ctypes); it exists so that the boundary is proven to bind where the reference's
  own shims (src/sampling.cpp:9-18 ...) would call it.
* ``blocks_aten.cpp`` IS the path of ``gated_ffn`` and ``residual_norm``: their checks, allocations and autograd nodes.
"""
import hashlib
import importlib.machinery
import importlib.util
import os

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
BUILD_DIR = os.path.join(HERE, "_build")
BLOCKS_DIR = os.path.join(BUILD_DIR, "blocks")
NAME = "butd_pointnet2_aten"
BLOCKS = "butd_blocks_aten"
FLAGS = ["-O2", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1"]


def _stamp(source):
    """What a front end is made of: its source, the headers of include/ that it names, the flags, torch."""
    import torch
    from .. import build as libbuild
    path = os.path.join(HERE, source)
    h = hashlib.sha1(" ".join(FLAGS + [torch.__version__]).encode())
    for p in [path] + libbuild._headers(path, []):
        with open(p, "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def _compile(name, source, directory, verbose):
    import torch  # noqa: F401
    from torch.utils import cpp_extension
    from .. import build as libbuild
    lib_path = libbuild.build()
    lib_dir = os.path.dirname(lib_path)
    os.makedirs(directory, exist_ok=True)
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    return cpp_extension.load(
        name=name, sources=[os.path.join(HERE, source)],
        extra_include_paths=[os.path.join(ROOT, "include"), os.path.join(rocm, "include")],
        extra_cflags=FLAGS,
        extra_ldflags=[f"-L{lib_dir}", "-lbutd_detr_hip", f"-Wl,-rpath,{lib_dir}",
                       f"-L{os.path.join(os.path.dirname(torch.__file__), 'lib')}", "-lc10_hip", "-ltorch_hip"],
        build_directory=directory, with_cuda=False, verbose=verbose)


def load(verbose=False):
    """Compile (first call) and import the reference's module surface."""
    return _compile(NAME, "pointnet2_aten.cpp", BUILD_DIR, verbose)


def compile_blocks(verbose=False):
    """Compile what changed of the blocks' front end and import it."""
    global _blocks
    stamp = _stamp("blocks_aten.cpp")
    _blocks = _compile(BLOCKS, "blocks_aten.cpp", BLOCKS_DIR, verbose)
    with open(os.path.join(BLOCKS_DIR, BLOCKS + ".stamp"), "w") as f:
        f.write(stamp)
    return _blocks


_blocks = None


def blocks():
    """The blocks' front end as it was built; compiled only where nothing is built yet.  RuntimeError where it was built from
    other sources: its argument structs may not be the library's."""
    global _blocks
    if _blocks is None:
        import torch
        path, stamp = os.path.join(BLOCKS_DIR, BLOCKS + ".so"), os.path.join(BLOCKS_DIR, BLOCKS + ".stamp")
        if not os.path.exists(path):
            if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{path} is not built and a graph is being captured: python -m butd_detr_amd.binding.build")
            return compile_blocks()
        built = open(stamp).read() if os.path.exists(stamp) else ""
        if built != _stamp("blocks_aten.cpp"):
            raise RuntimeError(f"{path} was built from other sources: build it with `python -m butd_detr_amd.binding.build`")
        from .. import _hiplib
        _hiplib.load()                         # (the library it links: missing -> says how to build it)
        spec = importlib.util.spec_from_file_location(BLOCKS, path, loader=importlib.machinery.ExtensionFileLoader(BLOCKS, path))
        _blocks = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_blocks)
    return _blocks


if __name__ == "__main__":
    for m in (load(verbose=True), compile_blocks(verbose=True)):
        print(m.__file__)
