class Optimizer:
    def __init__(self, parameters=None, lr=0.01, weight_decay=0.):
        self._parameters = parameters
        self.lr = lr
        self.weight_decay = weight_decay
        self.iterations = 0

    def zero_grad(self):
        for v in self._parameters:
            v.zero_grad()

    def step(self):
        self.iterations += 1
