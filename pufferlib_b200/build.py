"""In-tree build of the native libraries (sm_100a only).

Plays the part of the reference's `build_torch` step (setup.py:170-178,
237-258: CUDAExtension("pufferlib._C", [pufferlib.cpp, cuda/pufferlib.cu]) with
nvcc flags `-O3`), with the flags this implementation needs instead:

  libpuff_advantage_sm100.so   nvcc, -gencode arch=compute_100a,code=sm_100a,
                               no fast-math, no FTZ, no torch headers: the
                               kernels and their C ABI (include/puff_advantage.h)
  _C.so                        g++, torch headers: the TORCH_LIBRARY operator
                               registration, linked against the library above

Both land next to this file so that the package works from the source tree.
Outputs are rebuilt only when a source is newer or when they were made under
other settings (command, compiler, torch), which build/ keeps a record of.
"""
import hashlib
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

CUDA_HOME = os.environ.get("CUDA_HOME", "/usr/local/cuda")
NVCC = os.path.join(CUDA_HOME, "bin", "nvcc")

CABI_LIB = os.path.join(HERE, "libpuff_advantage_sm100.so")
TORCH_EXT = os.path.join(HERE, "_C.so")
OBJ_DIR = os.path.join(HERE, "build")   # object files, kept between builds

CU_SOURCES = ["puff_advantage_sm100.cu", "puff_priorities_sm100.cu", "puff_minibatch_sm100.cu",
              "puff_rollout_sm100.cu", "puff_host_pipeline.cu", "puff_logprobs_sm100.cu",
              "puff_policy_loss_sm100.cu", "puff_recurrence_sm100.cu"]
TORCH_SOURCES = ["torch_binding.cpp", "torch_policy_binding.cpp"]

# --fmad=true leaves nvcc free to contract a*b+c into an FMA.  One such contraction in the
# recurrence changes the last bit of about half of the outputs, so every kernel that must be
# bit-exact (tma2d, bulk1d, generic, and the replay step of scan) spells its arithmetic with
# __fmul_rn / __fadd_rn / __fsub_rn and their f32x2 forms, which are never contracted.  Only code
# that is checked against a tolerance (the scan kernel's carry composition, the minibatch
# normalisation, the priority weights) is written with plain operators and may be fused.
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "--ftz=false", "--prec-div=true", "--prec-sqrt=true", "--fmad=true",
    "-Xcompiler", "-fPIC", "-shared",
]


def _host_cxx():
    """The system g++.  A compiler wrapper that points the linker at a static
    libstdc++ (as the CXX of some build images does) would embed a second,
    uninitialised copy of the C++ runtime in the module; its iostreams crash
    the first time an error message formats a number."""
    override = os.environ.get("PUFF_CXX")
    if override:
        return override
    for cand in ("/usr/bin/g++", shutil.which("g++"), os.environ.get("CXX")):
        if cand and os.path.exists(cand):
            return cand
    return "g++"


def _settings(command, versions=()):
    """What decides about a compiled file besides its sources: the command, the
    compiler behind it and the versions of the libraries whose headers it reads.
    None without that compiler: then only the age of what is there can be looked at."""
    try:
        compiler = subprocess.run([command[0], "--version"], capture_output=True, text=True).stdout
    except OSError:
        return None
    return hashlib.sha256(repr([list(command), compiler, list(versions)]).encode()).hexdigest()


def _record_of(target):
    return os.path.join(OBJ_DIR, os.path.basename(target) + ".settings")


def _record(target, settings):
    os.makedirs(OBJ_DIR, exist_ok=True)
    with open(_record_of(target) + f".{os.getpid()}", "w") as f:
        f.write(settings)
    os.replace(f.name, _record_of(target))


def _stale(target, sources, settings=None):
    """Older than a source, or recorded as made under other settings."""
    if not os.path.isfile(target):
        return True
    if settings is not None and os.path.isfile(_record_of(target)):
        with open(_record_of(target)) as f:
            if f.read() != settings:
                return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def _link(command, target, rest, settings, verbose):
    """Under a name of its own first: a process that loads the library meanwhile, or another build, sees a whole one."""
    part = f"{target}.{os.getpid()}.part"
    try:
        _run(command + ["-o", part] + rest, verbose)
        os.replace(part, target)
    finally:
        if os.path.exists(part):
            os.remove(part)
    _record(target, settings)


def build_debug_cabi(out_path, verbose=False):
    """The kernel library with -DPUFF_DEBUG_BOUNDS: every global-memory index
    the kernels form is checked, a bad one sets PUFF_ERR_DEVICE_BOUNDS in the
    status word and its access is skipped (nothing traps).  Slower; for tests
    and debugging.  Written to `out_path`, never over the release library."""
    sources = [os.path.join(CSRC, s) for s in CU_SOURCES]
    _run([NVCC] + NVCC_FLAGS + ["-DPUFF_DEBUG_BOUNDS", "-o", out_path] + sources, verbose)
    return out_path


def _objects(sources, deps_of_all, command, force, verbose, versions=(), also=()):
    """Compile each source to build/<name>.<settings>.o unless that object is newer
    than the source and every file of `deps_of_all`; stale ones are compiled side by
    side.  `also`: flags that leave the object as it is (what the compiler prints)."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    settings = (_settings(command, versions) or "unknown")[:12]
    objects, running = [], []
    for name in sources:
        src, obj = os.path.join(CSRC, name), os.path.join(OBJ_DIR, f"{name}.{settings}.o")
        objects.append(obj)
        if force or _stale(obj, [src] + deps_of_all):
            part = f"{obj}.{os.getpid()}.part"
            cmd = command + list(also) + ["-c", "-o", part, src]
            if verbose:
                print(" ".join(cmd), flush=True)
            running.append((cmd, part, obj, subprocess.Popen(cmd)))
    failed = None
    for cmd, part, obj, proc in running:
        if proc.wait() == 0:
            os.replace(part, obj)
        else:
            failed = failed or cmd
            if os.path.exists(part):
                os.remove(part)
    if failed:
        raise subprocess.CalledProcessError(1, failed)
    for name in sources:        # objects of settings that are gone
        for old in os.listdir(OBJ_DIR):
            if old.startswith(name + ".") and old.endswith(".o") and os.path.join(OBJ_DIR, old) not in objects:
                os.remove(os.path.join(OBJ_DIR, old))
    return objects


def build_cabi(force=False, verbose=False, ptxas_info=False):
    headers = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith(".cuh")]
    headers.append(os.path.join(INCLUDE, "puff_advantage.h"))
    sources = [os.path.join(CSRC, s) for s in CU_SOURCES]
    settings = _settings([NVCC] + NVCC_FLAGS)
    if force or ptxas_info or _stale(CABI_LIB, sources + headers, settings):
        flags = [f for f in NVCC_FLAGS if f != "-shared"]
        objects = _objects(CU_SOURCES, headers, [NVCC] + flags, force or ptxas_info, verbose,
                           also=["-Xptxas", "-v"] if ptxas_info else [])
        _link([NVCC] + NVCC_FLAGS, CABI_LIB, objects, settings, verbose)
    return CABI_LIB


def build_torch_ext(force=False, verbose=False):
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    header = os.path.join(INCLUDE, "puff_advantage.h")
    deps = [os.path.join(CSRC, s) for s in TORCH_SOURCES] + [header, CABI_LIB]
    cxx = _host_cxx()
    inc = [f"-I{p}" for p in include_paths()]
    inc += [f"-I{os.path.join(CUDA_HOME, 'include')}", f"-I{sysconfig.get_paths()['include']}"]
    libdir = library_paths()[0]
    flags = [cxx, "-O2", "-std=c++17", "-fPIC",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             "-DTORCH_EXTENSION_NAME=_C"] + inc
    versions = [torch.__version__, torch.version.cuda]
    settings = _settings(flags, versions)
    if force or _stale(TORCH_EXT, deps, settings):
        objects = _objects(TORCH_SOURCES, [header], flags, force, verbose, versions)
        _link([cxx, "-shared"], TORCH_EXT, objects + [
              f"-L{HERE}", "-lpuff_advantage_sm100", "-Wl,-rpath,$ORIGIN",
              f"-L{libdir}", f"-Wl,-rpath,{libdir}",
              "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch"], settings, verbose)
    return TORCH_EXT


def build_all(force=False, verbose=False):
    build_cabi(force=force, verbose=verbose)
    build_torch_ext(force=force, verbose=verbose)


if __name__ == "__main__":
    if "--debug-bounds" in sys.argv:
        build_debug_cabi(os.path.join(HERE, "libpuff_advantage_sm100_debug.so"), verbose=True)
    else:
        build_all(force="--force" in sys.argv, verbose=True)
