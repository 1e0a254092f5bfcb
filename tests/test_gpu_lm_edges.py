"""The decoder's serving step where it is easily wrong: threads with batches of their own, scales and scores far apart, pages below a
window, numbers at the ends of their types, more work than a launch counts."""
import threading

import numpy as np
import pytest

from test_gpu_lm import Bed, to_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(gpx):
    c = gpx.LmContext()
    yield c
    assert c.status() == (0, 0)
    c.free()


# ---- threads ----------------------------------------------------------------------------------------

def test_threads_with_batches_of_their_own(gpx):
    """Two tenants in two threads, whose launches of the same kernels need different amounts of shared memory."""
    heads, kv, dim, page, dtype = 8, 2, 128, 64, "bfloat16"
    turn, wrong = [threading.Semaphore(1), threading.Semaphore(0)], []

    def tenant(me, seqs):
        try:
            gpx.init_cuda(0)
            mine, s = gpx.LmContext(), gpx.Stream(0)
            bed = Bed(gpx, [2] * seqs, [40 + 3 * i for i in range(seqs)], heads, kv, dim, page, seed=seqs).upload()
            x = gpx.DeviceBuffer.from_numpy(to_bits(bed.rng.standard_normal((bed.tokens, (heads + 2 * kv) * dim)), dtype))
            q, out = (gpx.DeviceBuffer(bed.tokens * heads * dim * 2) for _ in range(2))
            at, ld, want = x.ptr.value, (heads + 2 * kv) * dim, None

            def step():
                gpx.kv_append(bed.cache, bed.batch, at, at + 2 * heads * dim, at + 2 * (heads + kv) * dim, q, heads, dtype, mine, None, None, s, ld, ld, ld)
                gpx.kv_attend(bed.cache, bed.batch, q, out, heads, dtype, mine, stream=s)
                s.sync()
                return out.download(np.uint16, stream=s)

            for i in range(600):
                if i < 6:  # (in turn, then as it comes)
                    turn[me].acquire()
                try:
                    got = step()
                finally:
                    if i < 6:
                        turn[1 - me].release()
                if i == 1:
                    want = got  # (the second append finds the scales of the first)
                if i > 1 and not np.array_equal(got, want):
                    wrong.append(f"step {i} of {seqs} sequences")
                    break
            if mine.status() != (0, 0):
                wrong.append(f"status {mine.status()}")
            for b in (x, q, out, mine, bed):
                b.free()
            s.destroy()
        except Exception as e:  # noqa: BLE001
            wrong.append(repr(e))
            turn[1 - me].release(6)

    threads = [threading.Thread(target=tenant, args=a) for a in ((0, 64), (1, 8))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
