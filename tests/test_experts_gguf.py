"""The matrices of a layer of experts from GGUF files: 3-D tensors through the Python and the C++ reader, and the element order of
Q4_0 blocks."""
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

import cretif_amd as cri
import experts_ref as ref
from cretif_amd import quant
from gguf_writer import GGUFWriter, T_STR

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GGML_NAME = {"q8_0": "q8_0", "q4_0": "q4_0", "q5_0": "q5_0", "q4_k": "q4_k", "q6_k": "q6_k", "fp16": "f16"}
E, N, K = 3, 40, 512
NAME = "blk.%d.ffn_gate_exps.weight"


@pytest.fixture
def model(tmp_path):
    w, raws = GGUFWriter().add("general.architecture", T_STR, "llama"), {}
    for i, f in enumerate(GGML_NAME):
        raws[f] = quant.synthetic_weights(f, E * N, K, seed=90 + i)
        w.add_tensor(NAME % i, [K, N, E], GGML_NAME[f], raws[f])
    path = str(tmp_path / "m.gguf")
    w.write(path)
    return path, raws


def test_file_of_3d_tensors(model):
    path, raws = model
    with cri.GGUFFile(path) as g:
        for i, f in enumerate(GGML_NAME):
            info = g.tensor(g.find_tensor(NAME % i))
            assert info["dims"] == [K, N, E] and info["format"] == cri.FORMAT_IDS[f] and info["byte_size"] == raws[f].nbytes
            assert np.array_equal(g.tensor_bytes(g.find_tensor(NAME % i)), raws[f].view(np.uint8).reshape(-1))


@pytest.mark.gpu
def test_products_of_a_file(model):
    path, raws = model
    M, k = 5, 2
    ids = np.array([[0, 1], [2, 0], [1, 2], [2, 1], [0, 2]])
    off, pairs, _ = ref.group(ids, E)
    x = np.random.default_rng(1).standard_normal((M, K)).astype(np.float32)
    groups = cri.ExpertGroups(M, k, E)
    cri.group_experts(torch.from_numpy(ids.astype(np.int32)).cuda(), groups)
    with cri.GGUFFile(path) as g:
        for i, f in enumerate(GGML_NAME):
            at = g.find_tensor(NAME % i)
            info = g.tensor(at)
            raw = torch.empty(info["byte_size"], dtype=torch.uint8, device="cuda")
            g.upload(at, raw)
            k_, n_, e_ = info["dims"]
            w = cri.ExpertWeights(f, raw, e_, n_, k_)
            out = torch.empty(M * k, N, device="cuda")
            cri.expert_matmul(w, groups, torch.from_numpy(x).cuda(), out)
            v, mag = ref.weights(f, raws[f], E, N, K)
            for e in range(E):
                ref.check(out[off[e]:off[e + 1]], ref.Product(x[pairs[off[e]:off[e + 1]] // k], v[e], mag[e]), f)


def reordered(b):
    """Blocks [..., 18] of upstream's order (elements i and i + 16 in byte i) in the library's."""
    b = b.copy()
    q = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1)
    b[..., 2:] = q[..., 0::2] | q[..., 1::2] << 4
    return b


@pytest.mark.gpu
@pytest.mark.parametrize("upstream", [False, True])
def test_order_of_q4_0(upstream):
    """One-hot rows read single weights: element i from byte i / 2, and upstream's blocks once they are reordered."""
    e_, n_, k_ = 2, 3, 64
    rng = np.random.default_rng(5)
    blocks = rng.integers(0, 256, (e_, n_, k_ // 32, 18)).astype(np.uint8)
    blocks[..., :2] = np.array([1.0, 0.5], np.float16).view(np.uint8).reshape(2, 2)[rng.integers(0, 2, blocks.shape[:3])]
    d = np.ascontiguousarray(blocks[..., :2]).view(np.float16)[..., 0].astype(np.float64)
    b = blocks[..., 2:].astype(np.int64)
    if upstream:
        q = np.concatenate([b & 15, b >> 4], -1)
        blocks = reordered(blocks)
    else:
        q = np.stack([b & 15, b >> 4], -1).reshape(b.shape[:3] + (32,))
    want = (d[..., None] * (q - 8)).reshape(e_, n_, k_)
    w = cri.ExpertWeights("q4_0", torch.from_numpy(blocks.reshape(-1)).cuda(), e_, n_, k_)
    groups = cri.ExpertGroups(k_, e_, e_)
    cri.group_experts(torch.arange(e_, dtype=torch.int32, device="cuda").repeat(k_, 1).contiguous(), groups)
    out = torch.empty(k_ * e_, n_, device="cuda")
    cri.expert_matmul(w, groups, torch.eye(k_, device="cuda"), out)
    assert np.array_equal(ref.f64(out).reshape(e_, k_, n_), want.transpose(0, 2, 1))


# ---- the C++ reader ------------------------------------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not found")
    folder = tmp_path_factory.mktemp("cpp")
    out, libdir = str(folder / "experts_file_check"), os.path.join(ROOT, "cretif_amd")
    cmd = [cxx, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I",
           "/opt/rocm/include", os.path.join(ROOT, "tests", "cpp", "experts_file_check.cpp"), "-L", libdir, "-lcretif",
           "-Wl,-rpath," + libdir, "-L", "/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath,/opt/rocm/lib", "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    w = np.zeros((2, 3, 32), np.float16)
    for e in range(2):
        for n in range(3):
            w[e, n, n] = 4 * e + n + 1
    path = str(folder / "experts.gguf")
    GGUFWriter().add("general.architecture", T_STR, "llama").add_tensor("blk.0.ffn_gate_exps.weight", [32, 3, 2], "f16", w).write(path)
    return out, path


def test_reader_cpu(program):
    r = subprocess.run([program[0], "cpu", program[1]], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


@pytest.mark.gpu
def test_reader_gpu(program):
    r = subprocess.run([program[0], "gpu", program[1]], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
