"""Limits of the drafted-decoding operators that no ordinary call comes near,
and waits that run out."""

import ctypes
import threading

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import private_genomic_dnagpt_b200 as eng  # noqa: E402

from test_draft_gpu import AttentionArgs, Rows  # noqa: E402


@pytest.fixture(scope="module")
def cc():
    return eng.GenCryptoContext(eng.CCParams(ring_dim_log=10, limbs=3, dnum=1, seed=3))


def attention_workspace(cc, **sizes):
    """No pointer is looked at and nothing is launched."""
    a = AttentionArgs(**(dict(scale=1.0) | sizes))
    return eng.lib().ckks_draft_attention_workspace(cc.h, ctypes.byref(a))


@pytest.mark.parametrize("sizes,last,step", [
    # float32 heads of 256: 512 x 128 units of 8 rows, tiles of 16 keys and one entry for a unit's start;
    # 32767 entries a unit are the most
    (dict(dtype=2, batch=512, q_heads=16, kv_heads=1, head_dim=256, nodes=64), 32766 * 16 - 64, 16),
    # float32 heads of 64: 512 x 64 units of 16 rows, tiles of 64 keys
    (dict(dtype=2, batch=512, q_heads=16, kv_heads=1, head_dim=64, nodes=64), 65534 * 64 - 64, 64),
    # 16-bit heads of 64: 2^20 units, tiles of 128 keys, one more for the new keys and four entries for the start
    (dict(dtype=0, batch=1 << 20, q_heads=1, kv_heads=1, head_dim=64, nodes=64), 2042 * 128, 128)])
def test_attention_list_fits_32_bits(cc, sizes, last, step):
    """The kernels that divide a list of tiles need a workspace for the parts
    of units; from the first size on at which the list would pass 2^31 entries
    the call goes to the kernel without one, which here divides no keys."""
    assert attention_workspace(cc, capacity=last, **sizes) > 0
    assert attention_workspace(cc, capacity=last + 1, **sizes) == 0
    assert attention_workspace(cc, capacity=last + step, **sizes) == 0


def test_warps_that_meet_leave_together(cc):
    """The waits of the attention kernel's softmax warps: one thread whose wait
    runs out takes all warps out with it (none is left at the barrier where
    they meet), the fault is reported once and the context stays usable."""
    lib = eng.lib()
    assert lib.ckks_selftest_group_wait(cc.h, -1) == 0
    for starved in (0, 6):
        assert lib.ckks_selftest_group_wait(cc.h, starved) == 3
        assert b"gave up" in lib.ckks_last_error()
    assert lib.ckks_selftest_group_wait(cc.h, -1) == 0
    cc.Synchronize()


class AccumulateArgs(ctypes.Structure):
    """ckks_draft_accumulate_args of include/ckks_b200.h."""
    _fields_ = ([(n, ctypes.c_int32) for n in ("dtype", "batch", "q_heads", "kv_heads", "head_dim", "nodes", "capacity",
                                               "reserved")] + [("scale", ctypes.c_double)]
                + [(n, Rows) for n in ("q", "k_cache", "acc")]
                + [(n, ctypes.c_void_p) for n in ("lse", "lens", "path", "count")])


def test_contexts_of_two_threads_share_no_launch_setting():
    """Two host threads, each with a context and a stream of its own, whose
    calls of one kernel take different amounts of shared memory."""
    lib, calls = eng.lib(), 2000
    buf = torch.zeros(1 << 20, device="cuda")  # lengths, counts and parents of 0 among them
    outs = [torch.zeros(1 << 20, device="cuda") for _ in range(2)]
    failed = []

    def work(i):
        cc = eng.GenCryptoContext(eng.CCParams(ring_dim_log=10, limbs=3, dnum=1, seed=3))
        stream, at, out = torch.cuda.Stream(), buf.data_ptr(), outs[i].data_ptr()
        group, D = (64, 63) if i else (1, 33)
        acc = AccumulateArgs(dtype=0, batch=1, q_heads=group, kv_heads=1, head_dim=64, nodes=1, capacity=64, scale=1.0,
                             q=Rows(at, 1 << 14, 64, 64), k_cache=Rows(at, 4096, 4096, 64), acc=Rows(out, 64, 64, 0),
                             lse=at, lens=at, path=at, count=at)
        att = AttentionArgs(dtype=2, batch=1, q_heads=1, kv_heads=1, head_dim=D, nodes=1, capacity=1, scale=1.0,
                            lens=at, parents=at, lse=out, **{n: Rows(at, 64, 64, 64) for n in
                                                            ("q", "k_cache", "v_cache", "k_new", "v_new")},
                            out=Rows(out + 4096, 64, 64, 64))
        for _ in range(calls):
            for call, a in ((lib.ckks_draft_accumulate, acc), (lib.ckks_draft_attention, att)):
                if call(cc.h, ctypes.byref(a), stream.cuda_stream):
                    failed.append(lib.ckks_last_error())
                    return
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
