"""The tables of many sequences as a program on the host keeps them, one token after the other."""
import torch


class Tables:
    def __init__(self, sequences, width, pages, page_size):
        self.page, self.width = page_size, width
        self.rows, self.lens, self.held = [[-1] * width for _ in range(sequences)], [0] * sequences, [0] * sequences
        self.free, self.taken, self.given = list(range(pages)), 0, pages

    def has(self, i):
        return -(-self.lens[i] // self.page)

    def append(self, new, tokens):
        ends, positions, slots, missing = [0], [], [], 0
        for i, n in enumerate(new):
            n = min(max(n, 0), tokens - ends[-1])
            ends.append(ends[-1] + n)
            for position in range(self.lens[i], self.lens[i] + n):
                positions.append(position)
                column = position // self.page
                if column < self.width and column >= self.has(i) and self.taken < self.given:
                    self.rows[i][column] = self.free[self.taken % len(self.free)]
                    self.taken += 1
                    self.lens[i] = position + 1
                elif column < self.has(i):
                    self.lens[i] = position + 1
                else:
                    slots.append(-1)
                    missing += 1
                    continue
                slots.append(self.rows[i][column] * self.page + position % self.page)
        rest = tokens - len(slots)
        return {"ends": torch.tensor(ends, dtype=torch.int32), "lens": torch.tensor(self.lens, dtype=torch.int32), "positions": torch.tensor(positions + [0] * rest, dtype=torch.int64),
                "slots": torch.tensor(slots + [-1] * rest, dtype=torch.int64), "cursor": torch.tensor([self.taken, self.given]), "missing": torch.tensor([missing], dtype=torch.int32)}

    def release(self, done):
        there = self.given - self.taken
        for i, d in enumerate(done):
            if not d:
                continue
            for page in self.rows[i][self.held[i]:self.has(i)]:
                if there < len(self.free):
                    self.free[self.given % len(self.free)] = page
                    self.given += 1
                    there += 1
            self.lens[i] = self.held[i] = 0

    def fork(self, parent, common):
        of = list(self.lens)
        for i, p in enumerate(parent):
            if 0 <= p < len(parent) and p != i and parent[p] < 0 and of[i] == 0:
                pages = max(0, min(common[i], of[p])) // self.page
                self.rows[i][:pages] = self.rows[p][:pages]
                self.lens[i], self.held[i] = pages * self.page, pages
