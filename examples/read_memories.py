"""Questions answered from retrieved memories: retrieval, then one attention layer that reads them.

Each question retrieves memories (query_memory_fast). The memories' tokens (four projections of each embedding, stamped with
the memory's time and episode, placed by rank and by row and column of the four) are encoded, each within its own episode;
then the question's tokens and, one at a time, an answer's read all of them, weighted by score and age. The three
steps are the same calls: plan, store, attend. Run from the repository's root:

    python examples/read_memories.py
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

import mars_amd  # noqa: E402
from mars_amd import RetrievalConfig, corpus  # noqa: E402
from mars_amd.reader import DeviceArray, PagedCache, Reader  # noqa: E402

HEADS, KV_HEADS, DIM, PAGE, TOKENS = 12, 4, 64, 16, 4      # 12 heads of 64: the width of an embedding
MAX_PAGES, POOL = 24, 80                                    # a request's table row; pages of the cache


def project(x, w):
    """(tokens, 768) -> q, k, v of every token, float16."""
    y = (x @ w).astype(np.float16).reshape(len(x), HEADS + 2 * KV_HEADS, DIM)
    return np.split(y, [HEADS, HEADS + KV_HEADS], axis=1)


class Session:
    """One layer's cache with the tables of a batch of requests."""

    def __init__(self, requests):
        self.reader = Reader(HEADS, KV_HEADS, DIM, "float16", PAGE, rope_dim=DIM, rope_sections=(16, 8, 8))
        self.cache = PagedCache(DeviceArray((POOL, KV_HEADS, PAGE, DIM), "float16"), DeviceArray((POOL, KV_HEADS, DIM, PAGE), "float16"),
                                DeviceArray((POOL * PAGE,), "float32"), DeviceArray((POOL * PAGE,), "int32"))
        self.requests = requests
        self.table = DeviceArray.from_numpy(np.zeros((requests, MAX_PAGES), np.int32))
        self.free = DeviceArray.from_numpy(np.arange(POOL, dtype=np.int32))
        # what a step reads and what it writes, in turn
        self.lens = [DeviceArray.from_numpy(np.zeros(requests, np.int32)) for _ in range(2)]
        self.left = [DeviceArray.from_numpy(np.array([POOL], np.int32)) for _ in range(2)]
        # retrieval decays scores by exp(-lambda age); here every head forgets at a rate of its own
        self.decay = DeviceArray.from_numpy((corpus.DECAY_LAMBDA * 0.5 ** np.arange(HEADS)).astype(np.float32))
        self.steps = []

    def step(self, new_lens, q, k, v, places, times, episodes):
        """new_lens[r] new tokens of each request, in order; places (3, tokens): time, row, column. Returns the layer's output."""
        up = DeviceArray.from_numpy
        tokens = len(q)
        q, k, v = up(q), up(k), up(v)
        start, slots, pos = DeviceArray((self.requests + 1,), "int32"), DeviceArray((tokens,), "int64"), DeviceArray((tokens,), "int32")
        lens = DeviceArray((self.requests,), "int32")
        times, episodes = up(times.astype(np.float32)), up(episodes.astype(np.int32))
        self.reader.plan(up(np.asarray(new_lens, np.int32)), self.lens[0], self.table, self.free, self.left[0], q_start=start,
                         kv_lens=lens, slots=slots, positions=pos, free_count_out=self.left[1], next_lens=self.lens[1])
        self.reader.store(self.cache, q, k, v, up(places.astype(np.int32)), slots, times=times, episodes=episodes)
        out = DeviceArray((tokens, HEADS, DIM), "float16")
        self.reader.attend(self.cache, q, out, start, lens, self.table, cap=30.0, decay=self.decay, q_times=times,
                           q_episodes=episodes, max_new=int(max(new_lens)))
        self.lens.reverse()
        self.left.reverse()
        y = out.numpy()                                     # waits: every input above may go now
        self.steps.append(dict(new_lens=list(new_lens), q=q.numpy(), out=y, start=start.numpy(), lens=lens.numpy(),
                               table=self.table.numpy(), times=times.numpy(), episodes=episodes.numpy()))
        return y.reshape(tokens, -1).astype(np.float32)

    def end(self):
        self.reader.release(DeviceArray.from_numpy(np.ones(self.requests, np.int32)), self.lens[0], self.table, self.free, self.left[0])
        return int(self.left[0].numpy()[0])


def main(questions=3, nodes=2000, answer_tokens=4, seed=7, say=print):
    mars_amd.init(0)
    rng = np.random.default_rng(seed)
    c = corpus.nsn_graph(corpus.make_corpus(nodes, 768, seed=seed))
    dg = mars_amd.upload_to_device(mars_amd.MemoryGraph(c.num_nodes, c.dim, c.row_offsets, c.col_indices, c.embeddings, c.modalities, c.timestamps))
    mars_amd.upload_episode_ids(dg, c.episode_ids)
    ctx = mars_amd.create_query_context(c.num_nodes, c.dim, 64)
    w = (rng.standard_normal((768, (HEADS + 2 * KV_HEADS) * DIM)) / 16).astype(np.float32)
    spread = (rng.standard_normal((TOKENS, 768, 768)) / 28).astype(np.float32)
    try:
        asked = c.embeddings[corpus.pick_queries(c.modalities, questions, seed=seed)]
        found = [[r.node_id for r in mars_amd.query_memory_fast(dg, ctx, q, corpus.QUERY_TIME, RetrievalConfig(
            top_k=10, time_decay_lambda=corpus.DECAY_LAMBDA, max_results_returned=15 - i))] for i, q in enumerate(asked)]
        s = Session(questions)
        # the memories: oldest first, four tokens each
        ids = [sorted(f, key=lambda n: c.timestamps[n]) for f in found]
        flat = np.concatenate(ids)
        x = np.stack([c.embeddings[flat] @ m for m in spread], axis=1).reshape(-1, 768)
        rank = np.concatenate([np.arange(len(i)) for i in ids])
        four = np.tile(np.arange(TOKENS), len(flat))
        places = np.stack([np.repeat(rank, TOKENS), four // 2, four % 2])
        s.step([len(i) * TOKENS for i in ids], *project(x, w), places, np.repeat(c.timestamps[flat], TOKENS), np.repeat(c.episode_ids[flat], TOKENS))
        # the questions, of different lengths, then an answer token by token; both read every episode
        size = [5 + i for i in range(questions)]
        at = [len(i) for i in ids]
        x = np.concatenate([np.stack([asked[i] @ spread[t % TOKENS] for t in range(n)]) for i, n in enumerate(size)])
        for turn in range(answer_tokens + 1):
            place = np.concatenate([at[i] + np.arange(n) for i, n in enumerate(size)])
            total = int(sum(size))
            y = s.step(size, *project(x, w), np.stack([place] * 3), np.full(total, corpus.QUERY_TIME + turn), np.full(total, -1))
            at = [a + n for a, n in zip(at, size)]
            x = y[np.cumsum(size) - 1]                      # each request's last row is its next token
            size = [1] * questions
        say(f"{questions} questions over {[len(i) for i in ids]} memories: cached tokens {s.lens[0].numpy().tolist()}, pages in use "
            f"{POOL - int(s.left[0].numpy()[0])}")
        free = s.end()
        say(f"released: {free} of {POOL} pages free; |answer| {np.linalg.norm(x, axis=1).round(3).tolist()}")
        return s, free
    finally:
        mars_amd.destroy_query_context(ctx)
        mars_amd.free_device(dg)


if __name__ == "__main__":
    main()
