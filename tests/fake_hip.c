/* The HIP calls that a launch of phobos_hip makes, recorded instead of run: loaded before the
 * library, it takes their place in a process without a GPU.  A launch sleeps after it was
 * recorded, so that other threads' launches come between wherever nothing keeps them out. */
#include <pthread.h>
#include <stdint.h>
#include <string.h>
#include <unistd.h>

typedef struct {
    void *stream;
    char name[64];
    uint64_t thread;
} launch_t;

static launch_t launches[65536];
static int count;
static pthread_mutex_t mu = PTHREAD_MUTEX_INITIALIZER;
static char dummy[256];

int fake_count(void) { return count; }
const launch_t *fake_launch(int i) { return &launches[i]; }

int hipSetDevice(int d) { return d != 0; }
int hipGetDevice(int *d) { return *d = 0; }
int hipFree(void *p) { return p != 0; }
int hipGetSymbolAddress(void **p, const void *s) { return *p = dummy, s == 0; }
int hipModuleLoad(void **m, const char *path) { return *m = dummy, path == 0; }
int hipModuleUnload(void *m) { return m == 0; }
int hipModuleGetFunction(void **f, void *m, const char *name) {
    return *f = strdup(name), m == 0;
}
int hipStreamCreateWithFlags(void **s, unsigned flags) {
    static char streams[64][64];
    static int next;
    (void)flags;
    return *s = streams[next++], next > 64;
}
int hipStreamDestroy(void *s) { return s == 0; }
int hipStreamSynchronize(void *s) { return (void)s, 0; }
int hipStreamGetDevice(void *s, int *d) { return (void)s, *d = 0; }
int hipThreadExchangeStreamCaptureMode(int *mode) { return (void)mode, 0; }
int hipModuleLaunchKernel(void *f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned by,
                          unsigned bz, unsigned shmem, void *stream, void **args, void **extra) {
    (void)gx, (void)gy, (void)gz, (void)bx, (void)by, (void)bz, (void)shmem, (void)args, (void)extra;
    pthread_mutex_lock(&mu);
    const int i = count++;
    launches[i].stream = stream;
    strncpy(launches[i].name, f, sizeof launches[i].name - 1);
    launches[i].thread = (uint64_t)pthread_self();
    pthread_mutex_unlock(&mu);
    usleep(300);
    return 0;
}
